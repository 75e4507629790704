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
#include <algorithm>
#include <cstring>

#include "cc1d.h"
#include "cc1d_dispatch.cuh"

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

// ---- forward ----
// Team: one warp (several per block) when a group fits 32 * K * V columns,
// else the block.
template <typename T, int V, int K, bool GATE>
__global__ void __launch_bounds__(512) norm_fwd_kernel(const __grid_constant__ NormArgs a, int warp_teams) {
  __shared__ float2 buf[2][32];
  griddep_wait();
  const int nw = blockDim.x >> 5;
  const int team = warp_teams ? 32 : blockDim.x;
  const int t = warp_teams ? (threadIdx.x & 31) : threadIdx.x;
  const int grp = blockIdx.y;
  const i64 c0 = (i64)grp * a.gs;
  const i64 slot = warp_teams ? (i64)blockIdx.x * nw + (threadIdx.x >> 5) : blockIdx.x;
  const i64 step = warp_teams ? (i64)gridDim.x * nw : gridDim.x;
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = col_of<V>(k, team, t) + j;
      w[k][j] = c < a.gs ? param<T>(a.w, c0 + c, a.w_f32) : 0.f;
      b[k][j] = c < a.gs && a.b ? param<T>(a.b, c0 + c, a.w_f32) : 0.f;
    }
  }
  int ph = 0;
  for (i64 row = slot; row < a.rows; row += step) {
    float u[K][V], s[GATE ? K : 1][V];
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      load_cols<T, V>(a.x, row * a.xs + c0 + c, c < a.gs, u[k]);
      if (GATE) load_cols<T, V>(a.z, row * a.zs + c0 + c, c < a.gs, s[k]);
    }
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
      mu = team_sum(f2(sum, 0.f), !warp_teams, buf[ph], nw).x * a.inv;
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
    const float var = team_sum(f2(sq, 0.f), !warp_teams, buf[ph], nw).x * a.inv;
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
#pragma unroll
        for (int j = 0; j < V; ++j) {
          u[k][j] = fmaf(u[k][j] * r, w[k][j], b[k][j]);
          if (GATE && !a.gate_first) u[k][j] *= s[k][j];
        }
        store_cols<T, V>(a.y, row * a.ys + c0 + c, u[k]);
      }
    }
  }
}

// ---- backward ----
template <typename T, int V, int K, bool GATE>
__global__ void __launch_bounds__(512) norm_bwd_kernel(const __grid_constant__ NormArgs a, int warp_teams) {
  __shared__ float2 buf[2][32];
  griddep_wait();
  const int nw = blockDim.x >> 5;
  const int team = warp_teams ? 32 : blockDim.x;
  const int t = warp_teams ? (threadIdx.x & 31) : threadIdx.x;
  const int grp = blockIdx.y;
  const i64 c0 = (i64)grp * a.gs;
  const i64 slot = warp_teams ? (i64)blockIdx.x * nw + (threadIdx.x >> 5) : blockIdx.x;
  const i64 step = warp_teams ? (i64)gridDim.x * nw : gridDim.x;
  float w[K][V], dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = col_of<V>(k, team, t) + j;
      w[k][j] = c < a.gs ? param<T>(a.w, c0 + c, a.w_f32) : 0.f;
      dw[k][j] = db[k][j] = 0.f;
    }
  }
  int ph = 0;
  for (i64 row = slot; row < a.rows; row += step) {
    // h: the normalised values; g: dO * w; both in registers for the sums.
    float h[K][V], g[K][V], z[GATE ? K : 1][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      load_cols<T, V>(a.x, row * a.xs + c0 + c, c < a.gs, h[k]);
      load_cols<T, V>(a.dy, row * a.dys + c0 + c, c < a.gs, g[k]);
      if (GATE) load_cols<T, V>(a.z, row * a.zs + c0 + c, c < a.gs, z[k]);
    }
    const float r = a.rstd[row * a.groups + grp];
    const float mu = a.layer ? a.mean[row * a.groups + grp] : 0.f;
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = col_of<V>(k, team, t);
      if (c < a.gs) {
        float dz[V];
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
            const float o = fmaf(hh, w[k][j], a.b ? param<T>(a.b, c0 + c + j, a.w_f32) : 0.f);
            dz[j] = d * o * (sg * fmaf(z[k][j], 1.f - sg, 1.f));
            d *= si;
          }
          dw[k][j] = fmaf(d, hh, dw[k][j]);
          db[k][j] += d;
          const float gg = d * w[k][j];
          c1 = fmaf(gg, hh, c1);
          c2 += gg;
          g[k][j] = gg;
          // Gate first: x is needed again and h follows from it; else h is.
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
  if (slot >= a.slots) return;
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
  int threads, warp_teams;
  i64 blocks;        // per group
  int slots;
};

bool aligned(const void* p, i64 pitch, int esize) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (pitch * esize) % 16 == 0);
}

constexpr int kMaxTeam = 512;  // threads: 128 registers each at one block per SM

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
  bool vec = a->gs % wide == 0 && aligned(p->x, p->x_row_stride, es) && aligned(p->z, p->z_row_stride, es);
  vec = vec && (bwd ? aligned(p->dy, p->dy_row_stride, es) && aligned(p->dx, p->dx_row_stride, es) &&
                          aligned(p->dz, p->dz_row_stride, es)
                    : aligned(p->y, p->y_row_stride, es));
  plan->v = vec ? wide : 1;
  const i64 acc = ceil_div(a->gs, plan->v);  // accesses per row and array
  // Values per thread: up to 32 forward, 16 backward (it holds three arrays
  // and the two sums); the team grows with the group.
  const int most = std::max(1, (bwd ? 16 : 32) / plan->v);
  plan->k = 1;
  while (plan->k < std::min(most, 8) && acc > 32 * plan->k) plan->k *= 2;
  const i64 team = ceil_div(acc, plan->k);
  DeviceInfo dev;
  const cudaError_t e = device_info(&dev);
  const int sms = e == cudaSuccess ? dev.sms : 148;
  if (e != cudaSuccess) (void)cudaGetLastError();  // sizes may be asked for without a GPU
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
    // Teams walk rows: enough blocks to fill the SMs' threads once.
    const i64 fill = ceil_div((i64)sms * std::max(1, (bwd ? 1024 : 2048) / plan->threads), a->groups);
    plan->blocks = std::max<i64>(1, std::min<i64>(ceil_div(p->rows, per_block), fill));
    plan->slots = (int)(plan->blocks * per_block);
  }
  a->slots = plan->slots;
  return CC1D_OK;
}

size_t norm_workspace(const NormArgs& a, const NormPlan& plan) {
  return (size_t)plan.slots * a.dim * sizeof(float) * (a.b ? 2 : 1);
}

template <typename T, int V, int K>
cudaError_t launch_norm_k(const NormArgs& a, const NormPlan& pl, bool bwd, cudaStream_t s) {
  const dim3 grid((unsigned)pl.blocks, (unsigned)a.groups), block(pl.threads);
  if (bwd)
    return a.z ? launch_pdl(norm_bwd_kernel<T, V, K, true>, grid, block, 0, s, a, pl.warp_teams)
               : launch_pdl(norm_bwd_kernel<T, V, K, false>, grid, block, 0, s, a, pl.warp_teams);
  return a.z ? launch_pdl(norm_fwd_kernel<T, V, K, true>, grid, block, 0, s, a, pl.warp_teams)
             : launch_pdl(norm_fwd_kernel<T, V, K, false>, grid, block, 0, s, a, pl.warp_teams);
}

template <typename T, int V>
cudaError_t launch_norm_v(const NormArgs& a, const NormPlan& pl, bool bwd, cudaStream_t s) {
  switch (pl.k) {
    case 1: return launch_norm_k<T, V, 1>(a, pl, bwd, s);
    case 2: return launch_norm_k<T, V, 2>(a, pl, bwd, s);
    case 4:
      if constexpr (V <= 8) return launch_norm_k<T, V, 4>(a, pl, bwd, s);
      break;
    case 8:
      if constexpr (V <= 4) return launch_norm_k<T, V, 8>(a, pl, bwd, s);
      break;
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
