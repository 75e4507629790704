// Gated RMS / layer norm, forward and backward (sm_100a).
//
// Per group of gs adjacent columns of a row, with s = silu(z):
//   u = x s (gate first) or x;  mu = mean(u) (layer) or 0;  r = 1 / sqrt(mean((u - mu)^2) + eps)
//   h = (u - mu) r;  o = h w + b;  y = o (gate first or no gate) or o s
// and backward, with dO = dy (gate first or no gate) or dy s:
//   dw = sum dO h;  db = sum dO;  g = dO w;  du = r (g - h mean(g h) - [layer] mean(g))
//   gate first: dx = du s, dz = du x silu'(z);  else dx = du, dz = dy o silu'(z)
// Bound by memory: the forward reads x (and z) and writes y, the backward
// reads x, dy (and z) and writes dx (and dz), each once.  A group of a row is
// held in registers in fp32 while its sums are taken (two passes over the
// registers: the variance is that of the centred values), by a team of
// threads that walks rows with a fixed stride, so that weight and bias are
// read once per team and their gradients' sums stay in registers.
// Measured on 16384 rows of 5120 in bf16, gated: forward 91 us (5.5 TB/s, 86 %
// of a plain copy's rate), backward 185 (4.5 TB/s; two passes over a row, each
// with SiLU: issue slots 62 % busy).  A single row: 3.0 us,
// in groups of 640 2.1.
#include <algorithm>
#include <cstring>

#include "cc1d.h"
#include "cc1d_dispatch.cuh"
#include "cc1d_tma.cuh"

namespace cc1d {

namespace {

struct NormArgs {
  const void* x; i64 xs;
  const void* z; i64 zs;
  const void* w;
  const void* b;
  void* y; i64 ys;
  float* mean;
  float* rstd;
  const void* dy; i64 dys;
  void* dx; i64 dxs;
  void* dz; i64 dzs;
  float* part;      // [2][slots][dim]: shares of dweight and dbias
  i64 rows, dim;
  int gs, groups;
  int slots;        // teams per group of columns
  float eps, inv;   // inv = 1 / gs
  int layer, gate_first, w_f32;
};

// A parameter in the data's type or fp32.
template <typename T>
__device__ __forceinline__ float param(const void* p, i64 i, int f32) {
  return f32 ? static_cast<const float*>(p)[i] : Cvt<T>::f(static_cast<const T*>(p)[i]);
}

// V adjacent ones, by 16-byte loads (V > 1: the plan has checked the alignment).
template <typename T, int V>
__device__ __forceinline__ void load_params(const void* p, i64 i, int f32, float (&o)[V]) {
  if constexpr (V == 1) {
    o[0] = param<T>(p, i, f32);
  } else if (f32) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + j));
      o[j] = v.x, o[j + 1] = v.y, o[j + 2] = v.z, o[j + 3] = v.w;
    }
  } else {
    const Pack<T, V> pk = ld_pack<T, V>(static_cast<const T*>(p) + i);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = Cvt<T>::f(pk.v[j]);
  }
}

// Sums of two values over a team: WARPS == 0, a warp; else the whole block,
// through shared memory (two buffers in turn, so one barrier per sum).
__device__ __forceinline__ float2 team_sum(float2 v, bool block, float2* buf, int nw) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(kFull, v.x, o);
    v.y += __shfl_xor_sync(kFull, v.y, o);
  }
  if (!block) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) buf[warp] = v;
  __syncthreads();
  v = lane < nw ? buf[lane] : f2(0.f, 0.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(kFull, v.x, o);
    v.y += __shfl_xor_sync(kFull, v.y, o);
  }
  return v;
}

// One value, the warps' parts added up by every thread itself.
__device__ __forceinline__ float team_sum(float v, bool block, float* buf, int nw) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  if (!block) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) buf[warp] = v;
  __syncthreads();
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < nw; i += 4) {  // the buffer is 0 behind the last warp's part
    const float4 p = *reinterpret_cast<const float4*>(buf + i);
    sum.x += p.x, sum.y += p.y, sum.z += p.z, sum.w += p.w;
  }
  return (sum.x + sum.y) + (sum.z + sum.w);
}

// Where a thread's values lie: V adjacent columns at (k * team + t) * V, k < K.
template <int V>
__device__ __forceinline__ int col_of(int k, int team, int t) { return (k * team + t) * V; }

template <typename T, int V>
__device__ __forceinline__ void load_cols(const void* base, i64 off, bool ok, float (&o)[V]) {
  if (ok) {
    const Pack<T, V> pk = ld_pack<T, V>(static_cast<const T*>(base) + off);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = Cvt<T>::f(pk.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = 0.f;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_cols(void* base, i64 off, const float (&o)[V]) {
  Pack<T, V> pk;
#pragma unroll
  for (int j = 0; j < V; ++j) pk.v[j] = Cvt<T>::to(o[j]);
  st_pack<T, V>(static_cast<T*>(base) + off, pk);
}

// ---- rows through shared memory ----
// With more than a few rows per block, each row's arrays come by bulk copies
// into a ring of stages: a block then has the next rows' bytes on their way
// without holding them in registers.  A stage is free again at the barrier of
// its row's first sum, by when every thread has its values in registers.
struct Ring {
  unsigned char* base;
  uint64_t* full;
  int stages;
  unsigned bytes;      // of one array's row
  unsigned stage;      // of a stage
};

// A stage and its phase, counted along (the number of stages is no constant).
struct RingAt {
  unsigned s = 0, phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == (unsigned)stages) s = 0, phase ^= 1;
  }
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, unsigned bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The group's weight (and bias) into shared memory, once per block: a block
// reads them with every row, and with the ring next to it the L1 cache is too
// small to keep them.
template <typename T>
__device__ __forceinline__ unsigned char* stage_params(const NormArgs& a, i64 c0, unsigned char* to) {
  const int es = a.w_f32 ? 4 : (int)sizeof(T);
  const int n16 = a.gs * es / 16;
  const uint4* w = reinterpret_cast<const uint4*>(static_cast<const char*>(a.w) + c0 * es);
  const uint4* b = a.b ? reinterpret_cast<const uint4*>(static_cast<const char*>(a.b) + c0 * es) : nullptr;
  uint4* o = reinterpret_cast<uint4*>(to);
  for (int i = threadIdx.x; i < n16; i += blockDim.x) {
    o[i] = __ldg(w + i);
    if (b) o[n16 + i] = __ldg(b + i);
  }
  return to + a.gs * es;  // the bias
}

// V adjacent values at p (shared or global memory, 16-byte aligned) as V / 2
// pairs, and back.
template <typename T, int V>
__device__ __forceinline__ void get_pairs(const void* p, float2 (&o)[V / 2]) {
  const uint4 w = *static_cast<const uint4*>(p);
  if constexpr (sizeof(T) == 4) {
    o[0] = f2(__uint_as_float(w.x), __uint_as_float(w.y));
    o[1] = f2(__uint_as_float(w.z), __uint_as_float(w.w));
  } else {
    o[0] = Pair<T>::unpack(w.x);
    o[1] = Pair<T>::unpack(w.y);
    o[2] = Pair<T>::unpack(w.z);
    o[3] = Pair<T>::unpack(w.w);
  }
}

template <typename T, int V>
__device__ __forceinline__ void put_pairs(void* p, const float2 (&v)[V / 2]) {
  uint4 w;
  if constexpr (sizeof(T) == 4) {
    w = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  } else {
    w = make_uint4(Pair<T>::pack(v[0]), Pair<T>::pack(v[1]), Pair<T>::pack(v[2]), Pair<T>::pack(v[3]));
  }
  *static_cast<uint4*>(p) = w;
}

template <typename T, int V>
__device__ __forceinline__ void param_pairs(const unsigned char* p, int c, int f32, float2 (&o)[V / 2]) {
  if (sizeof(T) == 4 || f32) {
#pragma unroll
    for (int j = 0; j < V / 2; j += 2) {
      const float4 v = *reinterpret_cast<const float4*>(p + (c + 2 * j) * 4);
      o[j] = f2(v.x, v.y), o[j + 1] = f2(v.z, v.w);
    }
  } else {
    get_pairs<T, V>(p + c * sizeof(T), o);
  }
}

template <int ARRAYS>
__device__ __forceinline__ void ring_fill(const Ring& r, unsigned s, const void* const (&src)[ARRAYS]) {
  mbar_arrive_expect_tx(&r.full[s], r.bytes * ARRAYS);
#pragma unroll
  for (int i = 0; i < ARRAYS; ++i) bulk_load(r.base + s * r.stage + i * r.bytes, src[i], r.bytes, &r.full[s]);
}

__device__ __forceinline__ Ring ring_make(unsigned char* smem, int stages, unsigned bytes, int arrays) {
  Ring r{smem + 128, reinterpret_cast<uint64_t*>(smem), stages, bytes, bytes * arrays};
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&r.full[s], 1);
    fence_mbar_init();
  }
  __syncthreads();
  return r;
}

// ---- forward ----
// Team: one warp (several per block) when a group fits 32 * K * V columns,
// else the block.
template <typename T, int V, int K, bool GATE>
__global__ void __launch_bounds__(512) norm_fwd_kernel(const __grid_constant__ NormArgs a, int warp_teams, int) {
  __shared__ __align__(16) float buf[2][32];
  if (threadIdx.x < 64) buf[threadIdx.x >> 5][threadIdx.x & 31] = 0.f;
  griddep_wait();
  __syncthreads();
  const int nw = blockDim.x >> 5;
  const int team = warp_teams ? 32 : blockDim.x;
  const int t = warp_teams ? (threadIdx.x & 31) : threadIdx.x;
  const int grp = blockIdx.y;
  const i64 c0 = (i64)grp * a.gs;
  const i64 slot = warp_teams ? (i64)blockIdx.x * nw + (threadIdx.x >> 5) : blockIdx.x;
  const i64 step = warp_teams ? (i64)gridDim.x * nw : gridDim.x;
  int ph = 0;
  for (i64 row = slot; row < a.rows; row += step) {
    float u[K][V], s[GATE ? K : 1][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      load_cols<T, V>(a.x, row * a.xs + c0 + c, c < a.gs, u[k]);
      if (GATE) load_cols<T, V>(a.z, row * a.zs + c0 + c, c < a.gs, s[k]);
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (GATE) {
          s[k][j] = silu_f(s[k][j]);
          if (a.gate_first) u[k][j] *= s[k][j];
        }
        sum += u[k][j];
      }
    }
    float mu = 0.f;
    if (a.layer) {
      mu = team_sum(sum, !warp_teams, buf[ph], nw) * a.inv;
      ph ^= 1;
    }
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (col_of<V>(k, team, t) < a.gs) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          u[k][j] -= mu;
          sq = fmaf(u[k][j], u[k][j], sq);
        }
      }
    }
    const float var = team_sum(sq, !warp_teams, buf[ph], nw) * a.inv;
    ph ^= 1;
    const float r = 1.f / sqrtf(var + a.eps);
    if (t == 0) {
      if (a.rstd) a.rstd[row * a.groups + grp] = r;
      if (a.mean) a.mean[row * a.groups + grp] = mu;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      if (c < a.gs) {
        float w[V], b[V];
        load_params<T, V>(a.w, c0 + c, a.w_f32, w);
        if (a.b) load_params<T, V>(a.b, c0 + c, a.w_f32, b);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          u[k][j] = fmaf(u[k][j] * r, w[j], a.b ? b[j] : 0.f);
          if (GATE && !a.gate_first) u[k][j] *= s[k][j];
        }
        store_cols<T, V>(a.y, row * a.ys + c0 + c, u[k]);
      }
    }
  }
}

// The same with rows in the ring, in pairs (packed fp32 math).
template <typename T, int V, int K, bool GATE>
__global__ void __launch_bounds__(512, 2) norm_fwd_ring_kernel(const __grid_constant__ NormArgs a, int, int stages) {
  __shared__ __align__(16) float buf[2][32];
  extern __shared__ __align__(128) unsigned char smem[];
  if (threadIdx.x < 64) buf[threadIdx.x >> 5][threadIdx.x & 31] = 0.f;
  griddep_wait();
  const int nw = blockDim.x >> 5, team = blockDim.x, t = threadIdx.x;
  const int grp = blockIdx.y;
  const i64 c0 = (i64)grp * a.gs, step = gridDim.x;
  constexpr int kArrays = GATE ? 2 : 1;
  unsigned char* sw = smem + 128 + stages * (unsigned)(a.gs * sizeof(T) * kArrays);
  const unsigned char* sb = stage_params<T>(a, c0, sw);
  const Ring ring = ring_make(smem, stages, a.gs * sizeof(T), kArrays);
  auto fill = [&](i64 row, unsigned s) {
    if (row >= a.rows) return;
    const void* src[kArrays];
    src[0] = static_cast<const T*>(a.x) + row * a.xs + c0;
    if (GATE) src[kArrays - 1] = static_cast<const T*>(a.z) + row * a.zs + c0;
    ring_fill<kArrays>(ring, s, src);
  };
  if (t == 0)
    for (int n = 0; n < stages; ++n) fill(blockIdx.x + n * step, n);
  int ph = 0;
  RingAt at;
  for (i64 row = blockIdx.x; row < a.rows; row += step) {
    (void)mbar_wait(&ring.full[at.s], at.phase);
    const unsigned char* st = ring.base + at.s * ring.stage;
    float2 u[K][V / 2], s[GATE ? K : 1][V / 2];
    float2 sq = f2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      if (c < a.gs) {
        get_pairs<T, V>(st + c * sizeof(T), u[k]);
        if (GATE) get_pairs<T, V>(st + ring.bytes + c * sizeof(T), s[k]);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          if (GATE) s[k][j] = silu2(s[k][j]);
          if (GATE && a.gate_first) u[k][j] = mul2(u[k][j], s[k][j]);
        }
      }
    }
    float mu = 0.f;
    if (a.layer) {
      float2 sum = f2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (col_of<V>(k, team, t) < a.gs) {
#pragma unroll
          for (int j = 0; j < V / 2; ++j) sum = add2(sum, u[k][j]);
        }
      }
      mu = team_sum(sum.x + sum.y, true, buf[ph], nw) * a.inv;
      ph ^= 1;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (col_of<V>(k, team, t) < a.gs) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          if (a.layer) u[k][j] = add2(u[k][j], f2(-mu, -mu));
          sq = fma2(u[k][j], u[k][j], sq);
        }
      }
    }
    const float var = team_sum(sq.x + sq.y, true, buf[ph], nw) * a.inv;
    ph ^= 1;
    if (t == 0) fill(row + ring.stages * step, at.s);
    at.next(ring.stages);
    const float r = 1.f / sqrtf(var + a.eps);
    if (t == 0) {
      if (a.rstd) a.rstd[row * a.groups + grp] = r;
      if (a.mean) a.mean[row * a.groups + grp] = mu;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      if (c < a.gs) {
        float2 w[V / 2];
        param_pairs<T, V>(sw, c, a.w_f32, w);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) u[k][j] = mul2(mul2(u[k][j], f2(r, r)), w[j]);
        if (a.b) {
          float2 b[V / 2];
          param_pairs<T, V>(sb, c, a.w_f32, b);
#pragma unroll
          for (int j = 0; j < V / 2; ++j) u[k][j] = add2(u[k][j], b[j]);
        }
        if (GATE && !a.gate_first) {
#pragma unroll
          for (int j = 0; j < V / 2; ++j) u[k][j] = mul2(u[k][j], s[k][j]);
        }
        put_pairs<T, V>(static_cast<T*>(a.y) + row * a.ys + c0 + c, u[k]);
      }
    }
  }
}

// ---- backward ----
template <typename T, int V, int K, bool GATE>
__global__ void __launch_bounds__(512) norm_bwd_kernel(const __grid_constant__ NormArgs a, int warp_teams, int) {
  __shared__ float2 buf[2][32];
  griddep_wait();
  const int nw = blockDim.x >> 5;
  const int team = warp_teams ? 32 : blockDim.x;
  const int t = warp_teams ? (threadIdx.x & 31) : threadIdx.x;
  const int grp = blockIdx.y;
  const i64 c0 = (i64)grp * a.gs;
  const i64 slot = warp_teams ? (i64)blockIdx.x * nw + (threadIdx.x >> 5) : blockIdx.x;
  const i64 step = warp_teams ? (i64)gridDim.x * nw : gridDim.x;
  float dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) dw[k][j] = db[k][j] = 0.f;
  }
  int ph = 0;
  for (i64 row = slot; row < a.rows; row += step) {
    // h: the normalised values (gate first: x); g: dO * w; both in registers
    // for the second pass.
    float h[K][V], g[K][V], z[GATE ? K : 1][V];
    const float r = a.rstd[row * a.groups + grp];
    const float mu = a.layer ? a.mean[row * a.groups + grp] : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      load_cols<T, V>(a.x, row * a.xs + c0 + c, c < a.gs, h[k]);
      load_cols<T, V>(a.dy, row * a.dys + c0 + c, c < a.gs, g[k]);
      if (GATE) load_cols<T, V>(a.z, row * a.zs + c0 + c, c < a.gs, z[k]);
    }
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      if (c < a.gs) {
        float w[V], b[V], dz[V];
        load_params<T, V>(a.w, c0 + c, a.w_f32, w);
        if (GATE && !a.gate_first && a.b) load_params<T, V>(a.b, c0 + c, a.w_f32, b);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float u = h[k][j], d = g[k][j];
          float sg = 0.f, si = 0.f;
          if (GATE) {
            sg = sigmoid_f(z[k][j]);
            si = z[k][j] * sg;
          }
          if (GATE && a.gate_first) u *= si;
          const float hh = (u - mu) * r;
          if (GATE && !a.gate_first) {
            const float o = fmaf(hh, w[j], a.b ? b[j] : 0.f);
            dz[j] = d * o * (sg * fmaf(z[k][j], 1.f - sg, 1.f));
            d *= si;
          }
          dw[k][j] = fmaf(d, hh, dw[k][j]);
          if (a.b) db[k][j] += d;
          const float gg = d * w[j];
          c1 = fmaf(gg, hh, c1);
          c2 += gg;
          g[k][j] = gg;
          if (!(GATE && a.gate_first)) h[k][j] = hh;
        }
        if (GATE && !a.gate_first) store_cols<T, V>(a.dz, row * a.dzs + c0 + c, dz);
      }
    }
    const float2 m = team_sum(f2(c1, c2), !warp_teams, buf[ph], nw);
    ph ^= 1;
    const float m1 = m.x * a.inv, m2 = a.layer ? m.y * a.inv : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      if (c < a.gs) {
        float dx[V], dz[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (GATE && a.gate_first) {
            const float x = h[k][j], sg = sigmoid_f(z[k][j]), si = z[k][j] * sg;
            const float hh = (x * si - mu) * r;
            const float du = r * (g[k][j] - fmaf(hh, m1, m2));
            dx[j] = du * si;
            dz[j] = du * x * (sg * fmaf(z[k][j], 1.f - sg, 1.f));
          } else {
            dx[j] = r * (g[k][j] - fmaf(h[k][j], m1, m2));
          }
        }
        store_cols<T, V>(a.dx, row * a.dxs + c0 + c, dx);
        if (GATE && a.gate_first) store_cols<T, V>(a.dz, row * a.dzs + c0 + c, dz);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = col_of<V>(k, team, t) + j;
      if (c < a.gs) {
        a.part[slot * a.dim + c0 + c] = dw[k][j];
        if (a.b) a.part[((i64)a.slots + slot) * a.dim + c0 + c] = db[k][j];
      }
    }
  }
}

// The same with rows in the ring: the second pass reads them from there once
// more, so that only the sums over rows stay in registers and three blocks of
// 320 threads share an SM.  A row's stage is filled again at the next row's
// barrier.
template <typename T, int V, int K, bool GATE, bool BIAS>
__global__ void __launch_bounds__(512, 2) norm_bwd_ring_kernel(const __grid_constant__ NormArgs a, int, int stages) {
  __shared__ float2 buf[2][32];
  __shared__ __align__(16) float buf1[2][32];
  if (threadIdx.x < 64) buf1[threadIdx.x >> 5][threadIdx.x & 31] = 0.f;
  extern __shared__ __align__(128) unsigned char smem[];
  griddep_wait();
  const int nw = blockDim.x >> 5, team = blockDim.x, t = threadIdx.x;
  const int grp = blockIdx.y;
  const i64 c0 = (i64)grp * a.gs;
  constexpr int kArrays = GATE ? 3 : 2;
  unsigned char* sw = smem + 128 + stages * (unsigned)(a.gs * sizeof(T) * kArrays);
  const unsigned char* sb = stage_params<T>(a, c0, sw);
  const Ring ring = ring_make(smem, stages, a.gs * sizeof(T), kArrays);
  auto fill = [&](i64 row, unsigned s) {
    if (row >= a.rows) return;
    const void* src[kArrays];
    src[0] = static_cast<const T*>(a.x) + row * a.xs + c0;
    src[1] = static_cast<const T*>(a.dy) + row * a.dys + c0;
    if (GATE) src[kArrays - 1] = static_cast<const T*>(a.z) + row * a.zs + c0;
    ring_fill<kArrays>(ring, s, src);
  };
  if (t == 0)
    for (int n = 0; n < stages; ++n) fill(blockIdx.x + (i64)n * gridDim.x, n);
  __syncthreads();
  float2 dw[K][V / 2], db[BIAS ? K : 1][V / 2];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) dw[k][j] = db[BIAS ? k : 0][j] = f2(0.f, 0.f);
  }
  unsigned n = 0, last = 0;
  RingAt at;
  for (i64 row = blockIdx.x; row < a.rows; row += gridDim.x, ++n) {
    const float r = a.rstd[row * a.groups + grp];
    const float mu = a.layer ? a.mean[row * a.groups + grp] : 0.f;
    (void)mbar_wait(&ring.full[at.s], at.phase);
    const unsigned char* st = ring.base + at.s * ring.stage;
    float2 c1 = f2(0.f, 0.f), c2 = f2(0.f, 0.f);
    const float2 rr = f2(r, r), nmu = f2(-mu, -mu);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      if (c < a.gs) {
        float2 xs[V / 2], ds[V / 2], zs[V / 2], ws[V / 2];
        get_pairs<T, V>(st + c * sizeof(T), xs);
        get_pairs<T, V>(st + ring.bytes + c * sizeof(T), ds);
        if (GATE) get_pairs<T, V>(st + 2 * ring.bytes + c * sizeof(T), zs);
        param_pairs<T, V>(sw, c, a.w_f32, ws);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          float2 x = xs[j], d = ds[j];
          if (GATE) {
            const float2 si = silu2(zs[j]);
            if (a.gate_first)
              x = mul2(x, si);
            else
              d = mul2(d, si);
          }
          const float2 hh = mul2(add2(x, nmu), rr);
          dw[k][j] = fma2(d, hh, dw[k][j]);
          if (BIAS) db[BIAS ? k : 0][j] = add2(db[BIAS ? k : 0][j], d);
          const float2 g = mul2(d, ws[j]);
          c1 = fma2(g, hh, c1);
          if (a.layer) c2 = add2(c2, g);
        }
      }
    }
    const float2 m = a.layer ? team_sum(f2(c1.x + c1.y, c2.x + c2.y), true, buf[n & 1], nw)
                             : f2(team_sum(c1.x + c1.y, true, buf1[n & 1], nw), 0.f);
    if (t == 0 && n > 0) fill(row + (i64)(ring.stages - 1) * gridDim.x, last);
    last = at.s;
    at.next(ring.stages);
    const float2 m1 = f2(m.x * a.inv, m.x * a.inv), m2 = f2(m.y * a.inv, m.y * a.inv);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      if (c < a.gs) {
        float2 xs[V / 2], ds[V / 2], zs[V / 2], ws[V / 2], bs[V / 2];
        get_pairs<T, V>(st + c * sizeof(T), xs);
        get_pairs<T, V>(st + ring.bytes + c * sizeof(T), ds);
        if (GATE) get_pairs<T, V>(st + 2 * ring.bytes + c * sizeof(T), zs);
        param_pairs<T, V>(sw, c, a.w_f32, ws);
        if (BIAS && GATE && !a.gate_first) param_pairs<T, V>(sb, c, a.w_f32, bs);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          const float2 x = xs[j], d = ds[j], w = ws[j];
          float2 dx;
          if (GATE) {
            const float2 z = zs[j], one = f2(1.f, 1.f);
            const float2 sg = sigmoid2(z), si = mul2(z, sg), gr = mul2(sg, fma2(z, fma2(sg, f2(-1.f, -1.f), one), one));
            float2 dz;
            if (a.gate_first) {
              const float2 hh = mul2(add2(mul2(x, si), nmu), rr), tt = fma2(hh, m1, m2);
              const float2 du = mul2(rr, fma2(d, w, f2(-tt.x, -tt.y)));
              dz = mul2(mul2(du, x), gr);
              dx = mul2(du, si);
            } else {
              const float2 hh = mul2(add2(x, nmu), rr), tt = fma2(hh, m1, m2);
              dz = mul2(mul2(d, fma2(hh, w, BIAS ? bs[j] : f2(0.f, 0.f))), gr);
              dx = mul2(rr, fma2(mul2(d, si), w, f2(-tt.x, -tt.y)));
            }
            zs[j] = dz;
          } else {
            const float2 tt = fma2(mul2(add2(x, nmu), rr), m1, m2);
            dx = mul2(rr, fma2(d, w, f2(-tt.x, -tt.y)));
          }
          xs[j] = dx;
        }
        put_pairs<T, V>(static_cast<T*>(a.dx) + row * a.dxs + c0 + c, xs);
        if (GATE) put_pairs<T, V>(static_cast<T*>(a.dz) + row * a.dzs + c0 + c, zs);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = col_of<V>(k, team, t) + j;
      if (c < a.gs) {
        a.part[(i64)blockIdx.x * a.dim + c0 + c] = j % 2 ? dw[k][j / 2].y : dw[k][j / 2].x;
        if (BIAS) a.part[((i64)a.slots + blockIdx.x) * a.dim + c0 + c] = j % 2 ? db[BIAS ? k : 0][j / 2].y : db[BIAS ? k : 0][j / 2].x;
      }
    }
  }
}

// dweight and dbias from the teams' shares, in slot order: 8 warps of a
// block take every eighth slot of 32 columns, then add up through shared
// memory.  blockIdx.y: 0 dweight, 1 dbias.
template <typename T>
__global__ void norm_params_kernel(const float* part, i64 dim, int slots, void* dw, void* db, int w_f32) {
  __shared__ float sum[8][32];
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const i64 c = blockIdx.x * 32 + lane;
  const float* p = part + (i64)blockIdx.y * slots * dim;
  float v = 0.f;
  if (c < dim) {
#pragma unroll 8
    for (int s = warp; s < slots; s += 8) v += p[s * dim + c];
  }
  sum[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < dim) {
#pragma unroll
    for (int i = 1; i < 8; ++i) v += sum[i][lane];
    void* out = blockIdx.y ? db : dw;
    if (w_f32)
      static_cast<float*>(out)[c] = v;
    else
      static_cast<T*>(out)[c] = Cvt<T>::to(v);
  }
}

// ---- groups that no team's registers hold, and unaligned wide ones ----
// The row is read again for each pass (from L2); a block per (row, group).
template <typename T>
__global__ void __launch_bounds__(512) norm_wide_fwd_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float2 buf[2][32];
  griddep_wait();
  const int nw = blockDim.x >> 5;
  const i64 c0 = (i64)blockIdx.y * a.gs;
  for (i64 row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.xs + c0;
    const T* z = a.z ? static_cast<const T*>(a.z) + row * a.zs + c0 : nullptr;
    float sum = 0.f, mu = 0.f, sq = 0.f;
    auto val = [&](int c) {
      const float v = Cvt<T>::f(x[c]);
      return z && a.gate_first ? v * silu_f(Cvt<T>::f(z[c])) : v;
    };
    if (a.layer) {
      for (int c = threadIdx.x; c < a.gs; c += blockDim.x) sum += val(c);
      mu = team_sum(f2(sum, 0.f), true, buf[0], nw).x * a.inv;
    }
    for (int c = threadIdx.x; c < a.gs; c += blockDim.x) {
      const float v = val(c) - mu;
      sq = fmaf(v, v, sq);
    }
    const float r = 1.f / sqrtf(team_sum(f2(sq, 0.f), true, buf[1], nw).x * a.inv + a.eps);
    if (threadIdx.x == 0) {
      if (a.rstd) a.rstd[row * a.groups + blockIdx.y] = r;
      if (a.mean) a.mean[row * a.groups + blockIdx.y] = mu;
    }
    for (int c = threadIdx.x; c < a.gs; c += blockDim.x) {
      float v = fmaf((val(c) - mu) * r, param<T>(a.w, c0 + c, a.w_f32), a.b ? param<T>(a.b, c0 + c, a.w_f32) : 0.f);
      if (z && !a.gate_first) v *= silu_f(Cvt<T>::f(z[c]));
      static_cast<T*>(a.y)[row * a.ys + c0 + c] = Cvt<T>::to(v);
    }
    __syncthreads();
  }
}

// Backward of the same: a block walks its rows; the columns' sums are kept
// in its own slot of the workspace (each column by one thread, so no atomics).
template <typename T>
__global__ void __launch_bounds__(512) norm_wide_bwd_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float2 buf[32];
  griddep_wait();
  const int nw = blockDim.x >> 5;
  const i64 c0 = (i64)blockIdx.y * a.gs;
  float* pw = a.part + (i64)blockIdx.x * a.dim + c0;
  float* pb = a.part + ((i64)a.slots + blockIdx.x) * a.dim + c0;
  for (int c = threadIdx.x; c < a.gs; c += blockDim.x) {
    pw[c] = 0.f;
    if (a.b) pb[c] = 0.f;
  }
  for (i64 row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.xs + c0;
    const T* z = a.z ? static_cast<const T*>(a.z) + row * a.zs + c0 : nullptr;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dys + c0;
    const float r = a.rstd[row * a.groups + blockIdx.y];
    const float mu = a.layer ? a.mean[row * a.groups + blockIdx.y] : 0.f;
    float c1 = 0.f, c2 = 0.f;
    for (int c = threadIdx.x; c < a.gs; c += blockDim.x) {
      const float zv = z ? Cvt<T>::f(z[c]) : 0.f, si = silu_f(zv);
      const float u = Cvt<T>::f(x[c]) * (z && a.gate_first ? si : 1.f), hh = (u - mu) * r;
      const float d = Cvt<T>::f(dy[c]) * (z && !a.gate_first ? si : 1.f);
      pw[c] = fmaf(d, hh, pw[c]);
      if (a.b) pb[c] += d;
      const float g = d * param<T>(a.w, c0 + c, a.w_f32);
      c1 = fmaf(g, hh, c1);
      c2 += g;
    }
    const float2 m = team_sum(f2(c1, c2), true, buf, nw);
    const float m1 = m.x * a.inv, m2 = a.layer ? m.y * a.inv : 0.f;
    for (int c = threadIdx.x; c < a.gs; c += blockDim.x) {
      const float zv = z ? Cvt<T>::f(z[c]) : 0.f, si = silu_f(zv), xv = Cvt<T>::f(x[c]);
      const float hh = (xv * (z && a.gate_first ? si : 1.f) - mu) * r;
      const float dyv = Cvt<T>::f(dy[c]), wv = param<T>(a.w, c0 + c, a.w_f32);
      const float g = dyv * (z && !a.gate_first ? si : 1.f) * wv;
      const float du = r * (g - fmaf(hh, m1, m2));
      static_cast<T*>(a.dx)[row * a.dxs + c0 + c] = Cvt<T>::to(z && a.gate_first ? du * si : du);
      if (z) {
        const float gr = silu_grad_f(zv);
        const float o = fmaf(hh, wv, a.b ? param<T>(a.b, c0 + c, a.w_f32) : 0.f);
        static_cast<T*>(a.dz)[row * a.dzs + c0 + c] = Cvt<T>::to(a.gate_first ? du * xv * gr : dyv * o * gr);
      }
    }
    __syncthreads();
  }
}

// ---- host side ----

struct NormPlan {
  int v, k;          // columns per access, accesses per thread; k == 0: the wide kernels
  int stages;        // ring of rows; 0: none
  int threads, warp_teams;
  i64 blocks;        // per group
  unsigned smem;
  int slots;
};

bool aligned(const void* p, i64 pitch, int esize) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (pitch * esize) % 16 == 0);
}

constexpr int kMaxTeam = 512;

int plan_norm(const char* what, const cc1d_gated_norm_params* p, bool bwd, NormArgs* a, NormPlan* plan, bool* empty) {
  if (p == nullptr) return report_error(CC1D_ERR_INVALID_ARGUMENT, "%s: params is NULL", what);
  if (p->dtype != CC1D_F16 && p->dtype != CC1D_BF16 && p->dtype != CC1D_F32)
    return report_error(CC1D_ERR_UNSUPPORTED, "%s: unsupported dtype code %d", what, p->dtype);
  if (p->weight_dtype != p->dtype && p->weight_dtype != CC1D_F32)
    return report_error(CC1D_ERR_UNSUPPORTED, "%s: weight must be in the data's type or fp32", what);
  if (p->rows < 0 || p->dim < 0) return report_error(CC1D_ERR_INVALID_ARGUMENT, "%s: negative shape", what);
  *empty = p->dim == 0 || (p->rows == 0 && !bwd);
  if (*empty) return CC1D_OK;
  if (p->group_size < 1 || p->dim % p->group_size != 0)
    return report_error(CC1D_ERR_INVALID_ARGUMENT, "%s: dim (%lld) must be a multiple of group_size (%lld)", what,
                        (long long)p->dim, (long long)p->group_size);
  if (p->dim > 0x7fffffff / 2 || p->dim / p->group_size > 65535)
    return report_error(CC1D_ERR_UNSUPPORTED, "%s: dim is too large or has over 65535 groups", what);
  if (!p->weight || (p->rows > 0 && (!p->x || (!bwd && !p->y))) ||
      (bwd && (!p->dweight || (p->bias && !p->dbias) ||
               (p->rows > 0 && (!p->dy || !p->dx || !p->rstd || (p->layer && !p->mean) || (p->z && !p->dz))))))
    return report_error(CC1D_ERR_INVALID_ARGUMENT, "%s: a required tensor is missing", what);
  *a = NormArgs{p->x, p->x_row_stride, p->z, p->z_row_stride, p->weight, p->bias, p->y, p->y_row_stride,
                p->mean, p->rstd, p->dy, p->dy_row_stride, p->dx, p->dx_row_stride, p->dz, p->dz_row_stride,
                static_cast<float*>(p->workspace), p->rows, p->dim, (int)p->group_size, (int)(p->dim / p->group_size),
                0, p->eps, 1.f / (float)p->group_size, p->layer ? 1 : 0, p->gate_first ? 1 : 0,
                p->weight_dtype == CC1D_F32 ? 1 : 0};
  const int es = p->dtype == CC1D_F32 ? 4 : 2, wide = 16 / es;
  bool vec = a->gs % wide == 0 && aligned(p->weight, 0, es) && aligned(p->bias, 0, es) && aligned(p->x, p->x_row_stride, es) && aligned(p->z, p->z_row_stride, es);
  vec = vec && (bwd ? aligned(p->dy, p->dy_row_stride, es) && aligned(p->dx, p->dx_row_stride, es) &&
                          aligned(p->dz, p->dz_row_stride, es)
                    : aligned(p->y, p->y_row_stride, es));
  plan->v = vec ? wide : 1;
  const i64 acc = ceil_div(a->gs, plan->v);  // accesses per row and array
  // Values per thread: one vector (or four single ones) at first, up to 16
  // values where a warp can then hold the group, or where the team would pass
  // 512 threads.
  const int most = 16 / plan->v;
  plan->k = plan->v == 1 ? 4 : 1;
  while (plan->k < most && (acc > 512 * plan->k || (acc > 32 * plan->k && acc <= 64 * plan->k))) plan->k *= 2;
  const i64 team = ceil_div(acc, plan->k);
  DeviceInfo dev;
  const cudaError_t e = device_info(&dev);
  const int sms = e == cudaSuccess ? dev.sms : 148;
  if (e != cudaSuccess) (void)cudaGetLastError();  // sizes may be asked for without a GPU
  plan->stages = 0;
  if (team > kMaxTeam) {
    plan->k = 0;
    plan->threads = 512;
    plan->warp_teams = 0;
    plan->blocks = std::max<i64>(1, std::min<i64>(p->rows, ceil_div(sms * 4, a->groups)));
    plan->slots = (int)plan->blocks;
  } else {
    plan->warp_teams = team <= 32;
    plan->threads = plan->warp_teams ? 128 : (int)ceil_div(team, 32) * 32;
    const int per_block = plan->warp_teams ? 4 : 1;
    // Teams walk rows: blocks for as many threads as the registers hold.
    const int resident = std::max(1, 1024 / plan->threads);
    const unsigned stage = (unsigned)(a->gs * es) * ((bwd ? 2 : 1) + (p->z ? 1 : 0));
    if (!plan->warp_teams && vec) {
      // A ring where every resident block has a row, of 2 to 4 stages in what
      // shared memory these have.  Rows of 5120 in bf16, gated (ring | registers,
      // us): 148 rows 3.8 | 3.4, 444 rows 5.4 | 6.1, 1776 rows 12 | 16, 16384
      // rows 92 | 223; forward and backward 148 rows 14.0 | 12.7, 444 rows
      // 25 | 27, 16384 rows 271 | 626.
      const i64 fill = ceil_div((i64)sms * resident, a->groups);
      const int room = 220 * 1024 / resident;
      const int params = a->gs * (a->w_f32 ? 4 : es) * (p->bias ? 2 : 1);
      const int stages = std::min(4, (int)((room - 1024 - params) / (int)stage));
      if (stages >= 2 && p->rows >= fill) plan->stages = stages;
    }
    const i64 fill = ceil_div((i64)sms * resident, a->groups);
    plan->blocks = std::max<i64>(1, std::min<i64>(ceil_div(p->rows, per_block), fill));
    plan->slots = (int)(plan->blocks * per_block);
    plan->smem = plan->stages ? 128 + plan->stages * stage + a->gs * (a->w_f32 ? 4 : es) * (p->bias ? 2 : 1) : 0;
  }
  a->slots = plan->slots;
  return CC1D_OK;
}

size_t norm_workspace(const NormArgs& a, const NormPlan& plan) {
  return (size_t)plan.slots * a.dim * sizeof(float) * (a.b ? 2 : 1);
}

template <typename KERNEL>
cudaError_t launch_team(KERNEL kernel, std::atomic<uint64_t>& attr_done, const NormArgs& a, const NormPlan& pl, cudaStream_t s) {
  if (pl.smem > 48 * 1024) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev >= 0 && dev < 64 ? (1ull << dev) : 0ull;
    if (bit == 0 || !(attr_done.load(std::memory_order_acquire) & bit)) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 222 * 1024);
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
      if (e != cudaSuccess) return e;
      attr_done.fetch_or(bit, std::memory_order_acq_rel);
    }
  }
  return launch_pdl(kernel, dim3((unsigned)pl.blocks, (unsigned)a.groups), dim3(pl.threads), pl.smem, s, a, pl.warp_teams,
                    pl.stages);
}

template <typename T, int V, int K, bool GATE, bool RING>
cudaError_t launch_norm_k(const NormArgs& a, const NormPlan& pl, bool bwd, cudaStream_t s) {
  static std::atomic<uint64_t> fwd_done{0}, bwd_done{0}, bwd_bias_done{0};
  if constexpr (RING) {
    if (!bwd) return launch_team(norm_fwd_ring_kernel<T, V, K, GATE>, fwd_done, a, pl, s);
    return a.b ? launch_team(norm_bwd_ring_kernel<T, V, K, GATE, true>, bwd_bias_done, a, pl, s)
               : launch_team(norm_bwd_ring_kernel<T, V, K, GATE, false>, bwd_done, a, pl, s);
  } else {
    return bwd ? launch_team(norm_bwd_kernel<T, V, K, GATE>, bwd_done, a, pl, s)
               : launch_team(norm_fwd_kernel<T, V, K, GATE>, fwd_done, a, pl, s);
  }
}

template <typename T, int V, int K>
cudaError_t launch_norm_g(const NormArgs& a, const NormPlan& pl, bool bwd, cudaStream_t s) {
  if constexpr (V > 1) {
    if (pl.stages) return a.z ? launch_norm_k<T, V, K, true, true>(a, pl, bwd, s) : launch_norm_k<T, V, K, false, true>(a, pl, bwd, s);
  }
  return a.z ? launch_norm_k<T, V, K, true, false>(a, pl, bwd, s) : launch_norm_k<T, V, K, false, false>(a, pl, bwd, s);
}

template <typename T, int V>
cudaError_t launch_norm_v(const NormArgs& a, const NormPlan& pl, bool bwd, cudaStream_t s) {
  if constexpr (V == 1) {
    switch (pl.k) {
      case 4: return launch_norm_g<T, V, 4>(a, pl, bwd, s);
      case 8: return launch_norm_g<T, V, 8>(a, pl, bwd, s);
      case 16: return launch_norm_g<T, V, 16>(a, pl, bwd, s);
    }
  } else {
    switch (pl.k) {
      case 1: return launch_norm_g<T, V, 1>(a, pl, bwd, s);
      case 2: return launch_norm_g<T, V, 2>(a, pl, bwd, s);
      case 4:
        if constexpr (V <= 4) return launch_norm_g<T, V, 4>(a, pl, bwd, s);
        break;
    }
  }
  return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t launch_norm(const NormArgs& a, const NormPlan& pl, bool bwd, cudaStream_t s) {
  if (pl.k == 0) {
    const dim3 grid((unsigned)pl.blocks, (unsigned)a.groups), block(pl.threads);
    return bwd ? launch_pdl(norm_wide_bwd_kernel<T>, grid, block, 0, s, a)
               : launch_pdl(norm_wide_fwd_kernel<T>, grid, block, 0, s, a);
  }
  if (pl.v == 1) return launch_norm_v<T, 1>(a, pl, bwd, s);
  return launch_norm_v<T, 16 / (int)sizeof(T)>(a, pl, bwd, s);
}

template <typename T>
cudaError_t launch_params(const cc1d_gated_norm_params* p, const NormArgs& a, cudaStream_t s) {
  return launch_pdl(norm_params_kernel<T>, dim3((unsigned)ceil_div(a.dim, 32), a.b ? 2 : 1), dim3(256), 0, s,
                    (const float*)a.part, a.dim, a.slots, p->dweight, p->dbias, a.w_f32);
}

int norm_run(const char* what, const cc1d_gated_norm_params* p, bool bwd, void* stream) {
  NormArgs a;
  NormPlan pl;
  bool empty;
  // The plan needs the device's size: make the data's device current first.
  if (p != nullptr) {
    const void* ptr = bwd ? p->dweight : p->y;
    cudaPointerAttributes at;
    if (ptr != nullptr && cudaPointerGetAttributes(&at, ptr) == cudaSuccess && at.type == cudaMemoryTypeDevice && at.device >= 0) {
      int cur = -1;
      if (cudaGetDevice(&cur) == cudaSuccess && cur != at.device) {
        const cudaError_t e = cudaSetDevice(at.device);
        if (e != cudaSuccess) return report_cuda_error(e, what);
      }
    } else {
      (void)cudaGetLastError();
    }
  }
  const int rc = plan_norm(what, p, bwd, &a, &pl, &empty);
  if (rc != CC1D_OK || empty) return rc;
  const size_t need = bwd ? norm_workspace(a, pl) : 0;
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need))
    return report_error(CC1D_ERR_WORKSPACE, "%s: workspace of %zu bytes required", what, need);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = p->dtype == CC1D_F16    ? launch_norm<__half>(a, pl, bwd, s)
                  : p->dtype == CC1D_BF16 ? launch_norm<__nv_bfloat16>(a, pl, bwd, s)
                                          : launch_norm<float>(a, pl, bwd, s);
  if (e == cudaSuccess && bwd)
    e = p->dtype == CC1D_F16    ? launch_params<__half>(p, a, s)
        : p->dtype == CC1D_BF16 ? launch_params<__nv_bfloat16>(p, a, s)
                                : launch_params<float>(p, a, s);
  if (e != cudaSuccess) return report_cuda_error(e, what);
  return CC1D_OK;
}

}  // namespace

cudaError_t read_norm_wait_timeouts(unsigned* count) { return tu_read_wait_timeouts(count); }

}  // namespace cc1d

using namespace cc1d;

extern "C" int cc1d_gated_norm_fwd(const cc1d_gated_norm_params* p, void* stream) {
  return norm_run("cc1d_gated_norm_fwd", p, false, stream);
}

extern "C" int cc1d_gated_norm_workspace_size(const cc1d_gated_norm_params* p, size_t* bytes) {
  if (bytes == nullptr) return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_gated_norm_workspace_size: bytes is NULL");
  NormArgs a;
  NormPlan pl;
  bool empty = true;
  const int rc = plan_norm("cc1d_gated_norm_workspace_size", p, true, &a, &pl, &empty);
  *bytes = rc == CC1D_OK && !empty ? norm_workspace(a, pl) : 0;
  return rc;
}

extern "C" int cc1d_gated_norm_bwd(const cc1d_gated_norm_params* p, void* stream) {
  return norm_run("cc1d_gated_norm_bwd", p, true, stream);
}
