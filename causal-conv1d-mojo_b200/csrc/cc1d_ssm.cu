// Selective state space scan and its single-token step (sm_100a): the
// register-state kernels, the entry points and the choice of kernel.
//
// With S the (P, N) state of one head and sequence,
//   S_t = exp(dt_t A) S_{t-1} + dt_t x_t B_t^T,   y_t = S_t C_t + D x_t.
// The P rows of S are independent of one another given the token's B and C.
#include <algorithm>
#include <cstring>

#include "cc1d.h"
#include "cc1d_dispatch.cuh"
#include "cc1d_ssm.cuh"

namespace cc1d {

namespace {

constexpr int kMaxState = 256;  // dstate limit: 8 lanes of 32 state values

// Sums R values (one per row) over the 8 lanes of a row group; afterwards
// lane i of the group holds row i / (8 / R).
template <int R>
__device__ __forceinline__ float reduce_rows(const float (&acc)[R], int i) {
  float v;
  if constexpr (R == 4) {
    const bool hi = i & 4;
    const float k0 = (hi ? acc[2] : acc[0]) + __shfl_xor_sync(kFull, hi ? acc[0] : acc[2], 4);
    const float k1 = (hi ? acc[3] : acc[1]) + __shfl_xor_sync(kFull, hi ? acc[1] : acc[3], 4);
    const bool h2 = i & 2;
    v = (h2 ? k1 : k0) + __shfl_xor_sync(kFull, h2 ? k0 : k1, 2);
  } else if constexpr (R == 2) {
    const bool hi = i & 4;
    v = (hi ? acc[1] : acc[0]) + __shfl_xor_sync(kFull, hi ? acc[0] : acc[1], 4);
    v += __shfl_xor_sync(kFull, v, 2);
  } else {
    v = acc[0] + __shfl_xor_sync(kFull, acc[0], 4);
    v += __shfl_xor_sync(kFull, v, 2);
  }
  return v + __shfl_xor_sync(kFull, v, 1);
}

// ---- scan over tokens, the state in registers ----
//
// A warp owns 4 * R rows of one (sequence or segment, head): 8 lanes per
// row, VEC * NV state values each.  The block's 4 warps share a chunk of
// tokens that is staged in shared memory as fp32 (B, C, x, decay, step), so
// any type, stride and size works.  Per token and state value: one multiply,
// two fused multiply-adds.  Taken for fp32 data (the tensor cores would round
// it), for shapes the tensor-core kernel does not take, and for short sequences.
// Bound by the fp32 pipe on wide states (1.5 packed instructions per value)
// and the latency of a token's sums: 8 x 1024 fp32 tokens of 80 heads of
// 64 x 128 take 1001 us (1342 with scalar math and one chunk in flight);
// 2 x 512 of 4 heads of 16 x 16 take 14.5, in segments.
constexpr int kWalkThreads = 128;
// Tokens per staged chunk: as many as 48 KB of shared memory hold twice.
constexpr int walk_tokens(int np) { return np >= 256 ? 8 : np >= 64 ? 16 : 32; }

// 16 bytes from global to shared memory without registers, or zeros.
__device__ __forceinline__ void copy16(void* dst, const void* src, bool ok) {
  const unsigned d = static_cast<unsigned>(__cvta_generic_to_shared(dst)), n = ok ? 16u : 0u;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
}

// Rows [0, TOK) of a (tokens, n) operand into fp32 shared memory, zeros
// outside nt x n.  Of unit stride and 16-byte aligned rows, 16 bytes at a time
// (fp32: asynchronously, for the next wait_group); else element by element.
template <typename T, int TOK, int NP>
__device__ __forceinline__ void stage_rows(float (&to)[TOK][NP], const T* p, i64 ts, i64 ns, int nt, int n, bool wide) {
  constexpr int V = 16 / (int)sizeof(T);
  if (wide && NP % V == 0) {
    constexpr int W = NP >= V ? NP / V : 1;
    for (int e = threadIdx.x; e < TOK * W; e += kWalkThreads) {
      const int t = e / W, c = (e % W) * V;
      const bool ok = t < nt && c < n;
      const T* src = p + (ok ? t * ts + c : 0);
      if constexpr (sizeof(T) == 4) {
        copy16(&to[t][c], src, ok);
      } else {
        Pack<T, V> pk;
        if (ok) pk = ld_pack<T, V>(src);
#pragma unroll
        for (int j = 0; j < V; ++j) to[t][c + j] = ok ? Cvt<T>::f(pk.v[j]) : 0.f;
      }
    }
  } else {
    for (int e = threadIdx.x; e < TOK * NP; e += kWalkThreads) {
      const int t = e / NP, c = e % NP;
      to[t][c] = t < nt && c < n ? Cvt<T>::f(p[t * ts + c * ns]) : 0.f;
    }
  }
}

// Whether rows of n values can be read 16 bytes at a time.
template <typename T>
__device__ __forceinline__ bool wide_rows(const T* p, i64 ts, i64 ns, int n) {
  constexpr int V = 16 / (int)sizeof(T);
  return ns == 1 && n % V == 0 && ts % V == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

template <typename T, int VEC, int NV, int R, bool PART>
__global__ void __launch_bounds__(kWalkThreads) scan_walk_kernel(const __grid_constant__ ScanArgs a) {
  constexpr int NP = 8 * VEC * NV;   // padded state size
  constexpr int ROWS = 16 * R;       // rows per block
  constexpr int kWalkTokens = walk_tokens(NP);
  __shared__ __align__(16) float sB[2][kWalkTokens][NP];
  __shared__ __align__(16) float sC[2][PART ? 1 : kWalkTokens][NP];
  __shared__ __align__(16) float sx[2][kWalkTokens][ROWS];
  __shared__ float sw[2][kWalkTokens], sd[2][kWalkTokens];  // decay and step
  __shared__ float sl[2][PART ? kWalkTokens : 1];           // log of the decay
  griddep_wait();
  const int h = blockIdx.x % a.H;
  const i64 item = blockIdx.x / a.H;
  ScanItem it;
  if (!scan_locate(a, item, &it)) return;
  if (PART && it.seg + 1 >= it.nsegs) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, i = lane & 7;
  const int row_b = blockIdx.y * ROWS;                     // first row of the block
  const int row_w = warp * 4 * R + (lane >> 3) * R;        // this lane group's first row within it
  const int g = h / a.R;
  auto state_at = [&](int v) { return ((v / VEC) * 8 + i) * VEC + v % VEC; };  // this lane's v-th state value
  const float A = a.A[h];
  const float bias = a.dt_bias ? a.dt_bias[h] : 0.f;
  const float Dh = a.D ? a.D[h] : 0.f;
  const T* x = static_cast<const T*>(a.x) + it.batch * a.xs_b + h * a.xs_h;
  const T* Bp = static_cast<const T*>(a.B) + it.batch * a.bs_b + g * a.bs_g;
  const T* Cp = static_cast<const T*>(a.C) + it.batch * a.cs_b + g * a.cs_g;
  const i64 dto = it.batch * a.ds_b + h * a.ds_h;
  T* y = static_cast<T*>(a.y) + it.batch * a.ys_b + h * a.ys_h;

  float2 S[R][NV * VEC / 2];  // pairs along the state size: packed fp32 math
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int row = row_b + row_w + k;
#pragma unroll
    for (int v = 0; v < NV * VEC; ++v) {
      const int n = state_at(v);
      float s = 0.f;
      if (!PART && row < a.P && n < a.N) {
        const i64 e = (i64)row * a.N + n;
        if (a.init) {
          const i64 o = it.seq * a.is_s + h * a.is_h + e;
          s = a.init_f32 ? static_cast<const float*>(a.init)[o] : Cvt<T>::f(static_cast<const T*>(a.init)[o]);
        }
        for (int r = 0; r < it.seg; ++r) {  // the earlier segments, in order
          const i64 slot = (it.first + r) * a.H + h;
          s = fmaf(s, expf(a.decay[slot]), a.part[slot * a.P * a.N + e]);
        }
      }
      if (v % 2)
        S[k][v / 2].y = s;
      else
        S[k][v / 2].x = s;
    }
  }
  float total = 0.f;  // log of the segment's decay
  const bool wideB = wide_rows(Bp, a.bs_t, a.bs_n, a.N), wideC = wide_rows(Cp, a.cs_t, a.cs_n, a.N);
  const int rows = min(a.P - row_b, ROWS);
  const bool widex = wide_rows(x + row_b * a.xs_p, a.xs_t, a.xs_p, rows);
  // dt of this thread's token of a chunk, asked for a chunk ahead.
  auto raw_step = [&](i64 t0) {
    return tid < kWalkTokens && t0 + tid < it.t1 ? scan_raw_step<T>(a, dto + (t0 + tid) * a.ds_t) : 0.f;
  };
  float raw = raw_step(it.t0);
  auto stage = [&](int buf, i64 t0) {
    const int nt = (int)min((i64)kWalkTokens, it.t1 - t0);
    stage_rows<T>(sB[buf], Bp + t0 * a.bs_t, a.bs_t, a.bs_n, nt, a.N, wideB);
    if constexpr (!PART) stage_rows<T>(sC[buf], Cp + t0 * a.cs_t, a.cs_t, a.cs_n, nt, a.N, wideC);
    stage_rows<T>(sx[buf], x + t0 * a.xs_t + row_b * a.xs_p, a.xs_t, a.xs_p, nt, rows, widex);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (tid < nt) {
      const float v = raw + bias, d = a.softplus ? softplus_f(v) : v;
      sd[buf][tid] = d;
      // Accurate to the last bit or two: a state multiplies hundreds of these,
      // and the error of an approximate exponential (always to one side for one
      // step length) would add up to several times the rounding of fp32.
      sw[buf][tid] = expf(d * A);
      if (PART) sl[buf][tid] = d * A;
    }
    raw = raw_step(t0 + kWalkTokens);
  };
  if (it.t0 < it.t1) stage(0, it.t0);
  int buf = 0;
  for (i64 t0 = it.t0; t0 < it.t1; t0 += kWalkTokens, buf ^= 1) {
    const int nt = (int)min((i64)kWalkTokens, it.t1 - t0);
    // The next chunk is on its way while this one is worked on.
    if (t0 + kWalkTokens < it.t1) {
      stage(buf ^ 1, t0 + kWalkTokens);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
#pragma unroll 2
    for (int t = 0; t < nt; ++t) {
      const float d = sd[buf][t], w = sw[buf][t];
      if (PART) total += sl[buf][t];
      const float2 ww = f2(w, w);
      float2 u[R], sum[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const float ux = d * sx[buf][t][row_w + k];
        u[k] = f2(ux, ux);
        sum[k] = f2(0.f, 0.f);
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float2 b[VEC / 2], c[VEC / 2];
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) b[j] = *reinterpret_cast<const float2*>(&sB[buf][t][(v * 8 + i) * VEC + 2 * j]);
        if (!PART) {
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) c[j] = *reinterpret_cast<const float2*>(&sC[buf][t][(v * 8 + i) * VEC + 2 * j]);
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) {
            float2& s = S[k][v * VEC / 2 + j];
            s = fma2(s, ww, mul2(u[k], b[j]));
            if (!PART) sum[k] = fma2(s, c[j], sum[k]);
          }
        }
      }
      if (!PART) {
        float acc[R];
#pragma unroll
        for (int k = 0; k < R; ++k) acc[k] = sum[k].x + sum[k].y;
        const float v = reduce_rows<R>(acc, i);
        const int r = row_w + i / (8 / R);
        if ((i & (8 / R - 1)) == 0 && row_b + r < a.P)
          y[(t0 + t) * a.ys_t + row_b + r] = Cvt<T>::to(fmaf(Dh, sx[buf][t][r], v));
      }
    }
    __syncthreads();
  }
  float* out = nullptr;
  if (PART) {
    const i64 slot = item * a.H + h;
    out = a.part + slot * a.P * a.N;
    if (tid == 0 && blockIdx.y == 0) a.decay[slot] = total;
  } else if (a.fin && it.seg + 1 == it.nsegs) {
    out = a.fin + it.seq * a.fs_s + h * a.fs_h;
  }
  if (out == nullptr) return;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int row = row_b + row_w + k;
#pragma unroll
    for (int v = 0; v < NV * VEC; ++v) {
      const int n = state_at(v);
      if (row < a.P && n < a.N) out[(i64)row * a.N + n] = v % 2 ? S[k][v / 2].y : S[k][v / 2].x;
    }
  }
}

// y of the tokens outside every packed sequence.
template <typename T>
__global__ void scan_outside_kernel(const __grid_constant__ ScanArgs a) {
  griddep_wait();
  const i64 lo = min(max((i64)a.cu[0], (i64)0), a.L), hi = min(max((i64)a.cu[a.nseq], lo), a.L);
  const i64 gone = lo + (a.L - hi);
  const i64 cells = (i64)a.H * a.P;
  for (i64 e = blockIdx.x * (i64)blockDim.x + threadIdx.x; e < gone * cells; e += (i64)gridDim.x * blockDim.x) {
    const i64 r = e / cells;
    const int c = (int)(e - r * cells);
    const i64 t = r < lo ? r : hi + (r - lo);
    static_cast<T*>(a.y)[t * a.ys_t + (c / a.P) * a.ys_h + c % a.P] = Cvt<T>::to(0.f);
  }
}

template <typename T, int VEC, int NV, int R>
cudaError_t launch_walk_r(const ScanArgs& a, bool split, cudaStream_t stream) {
  const dim3 grid((unsigned)(a.items * a.H), (unsigned)ceil_div(a.P, 16 * R));
  if (split) {
    const cudaError_t e = launch_pdl(scan_walk_kernel<T, VEC, NV, R, true>, grid, dim3(kWalkThreads), 0, stream, a);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(scan_walk_kernel<T, VEC, NV, R, false>, grid, dim3(kWalkThreads), 0, stream, a);
}

// Rows per lane group: as many as the registers hold; one when P is small.
template <typename T, int VEC, int NV>
cudaError_t launch_walk_n(const ScanArgs& a, bool split, cudaStream_t stream) {
  if (VEC * NV <= 16 && a.P > 16) return launch_walk_r<T, VEC, NV, (VEC * NV <= 16 ? 4 : 1)>(a, split, stream);
  if (VEC * NV == 32 && a.P > 16) return launch_walk_r<T, VEC, NV, 2>(a, split, stream);
  return launch_walk_r<T, VEC, NV, 1>(a, split, stream);
}

template <typename T>
cudaError_t launch_walk(const ScanArgs& a, bool split, cudaStream_t stream) {
  if (a.N <= 16) return launch_walk_n<T, 2, 1>(a, split, stream);
  if (a.N <= 32) return launch_walk_n<T, 4, 1>(a, split, stream);
  if (a.N <= 64) return launch_walk_n<T, 4, 2>(a, split, stream);
  if (a.N <= 128) return launch_walk_n<T, 4, 4>(a, split, stream);
  return launch_walk_n<T, 4, 8>(a, split, stream);
}

// ---- one token per row, the state in memory ----
//
// Bound by the state's bytes (read once, written once); the rest is a few
// hundred values per head.  Eight lanes share a state row, as above, with VEC
// values (16 bytes where the layout allows) per access; a thread issues the
// loads of all its R rows before it uses one, and loads and stores are marked
// evict-first.  256 rows of 80 heads of 64 x 128 in fp32: 213 us, 6.3 TB/s;
// with ordinary accesses 239, with 4 rows per thread 250, with one 259.  Two
// are also sooner on few blocks (one row 3.9 | 4.0 us, 8 rows 8.1 | 10.4).
struct UpdArgs {
  const void* x; i64 xs_b, xs_h, xs_p;
  const void* dt; i64 ds_b, ds_h;
  const void* B; i64 bs_b, bs_g, bs_n;
  const void* C; i64 cs_b, cs_g, cs_n;
  const float* A;
  const float* D;
  const float* dt_bias;
  void* state; i64 ss_r, ss_h, ss_p;
  const int* idx;
  const int* oidx;
  void* y; i64 ys_b, ys_h;
  i64 rows;
  int H, P, N, R;
  int softplus, dt_f32;
};

template <typename T, typename ST, int VEC, int NV, int R>
__global__ void __launch_bounds__(128) scan_update_kernel(const __grid_constant__ UpdArgs a) {
  griddep_wait();
  const int h = blockIdx.x % a.H;
  const i64 b = blockIdx.x / a.H;
  const int lane = threadIdx.x & 31, i = lane & 7;
  const int row0 = blockIdx.y * 16 * R + ((threadIdx.x >> 5) * 4 + (lane >> 3)) * R;
  const int g = h / a.R;
  const i64 src = a.idx ? (i64)a.idx[b] : b;
  T* y = static_cast<T*>(a.y) + b * a.ys_b + h * a.ys_h;
  if (src < 0 || src >= a.rows) {  // an idle slot
    if ((i & (8 / R - 1)) == 0) {
      const int row = row0 + i / (8 / R);
      if (row < a.P) y[row] = Cvt<T>::to(0.f);
    }
    return;
  }
  const i64 dst = a.oidx ? (i64)a.oidx[b] : src;
  const bool keep = dst >= 0 && dst < a.rows;
  const ST* sp = static_cast<const ST*>(a.state) + src * a.ss_r + h * a.ss_h;
  ST* dp = static_cast<ST*>(a.state) + dst * a.ss_r + h * a.ss_h;

  Pack<ST, VEC> s[R][NV];
#pragma unroll
  for (int k = 0; k < R; ++k) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int n = (v * 8 + i) * VEC;
      if (row0 + k < a.P && n < a.N)
        s[k][v].raw = __ldcs(reinterpret_cast<const typename Pack<ST, VEC>::Raw*>(sp + (row0 + k) * a.ss_p + n));
      else
        s[k][v].raw = typename Pack<ST, VEC>::Raw();
    }
  }
  const i64 dto = b * a.ds_b + h * a.ds_h;
  float d = a.dt_f32 ? static_cast<const float*>(a.dt)[dto] : Cvt<T>::f(static_cast<const T*>(a.dt)[dto]);
  if (a.dt_bias) d += a.dt_bias[h];
  if (a.softplus) d = softplus_f(d);
  const float w = expf(d * a.A[h]);  // accurate: a decode multiplies thousands of these
  const float Dh = a.D ? a.D[h] : 0.f;
  float u[R], xr[R], acc[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    xr[k] = row0 + k < a.P ? Cvt<T>::f(static_cast<const T*>(a.x)[b * a.xs_b + h * a.xs_h + (row0 + k) * a.xs_p]) : 0.f;
    u[k] = d * xr[k];
    acc[k] = 0.f;
  }
  const T* Bp = static_cast<const T*>(a.B) + b * a.bs_b + g * a.bs_g;
  const T* Cp = static_cast<const T*>(a.C) + b * a.cs_b + g * a.cs_g;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int n = (v * 8 + i) * VEC;
    float bv[VEC], cv[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      bv[j] = n + j < a.N ? Cvt<T>::f(Bp[(n + j) * a.bs_n]) : 0.f;
      cv[j] = n + j < a.N ? Cvt<T>::f(Cp[(n + j) * a.cs_n]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      Pack<ST, VEC> o;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float t = fmaf(Cvt<ST>::f(s[k][v].v[j]), w, u[k] * bv[j]);
        acc[k] = fmaf(t, cv[j], acc[k]);  // y sees the state before it is rounded to its stored type
        o.v[j] = Cvt<ST>::to(t);
      }
      if (keep && row0 + k < a.P && n < a.N)
        __stcs(reinterpret_cast<typename Pack<ST, VEC>::Raw*>(dp + (row0 + k) * a.ss_p + n), o.raw);
    }
  }
  const float v = reduce_rows<R>(acc, i);
  const int k = i / (8 / R);
  float xk = xr[0];
#pragma unroll
  for (int q = 1; q < R; ++q) xk = k == q ? xr[q] : xk;
  if ((i & (8 / R - 1)) == 0 && row0 + k < a.P) y[row0 + k] = Cvt<T>::to(fmaf(Dh, xk, v));
}

template <typename T, typename ST, int VEC, int NV>
cudaError_t launch_upd_n(const UpdArgs& a, i64 batch, cudaStream_t stream) {
  constexpr int R = NV * VEC <= 32 ? 2 : 1;
  if (a.P > 16) {
    const dim3 grid((unsigned)(batch * a.H), (unsigned)ceil_div(a.P, 16 * R));
    return launch_pdl(scan_update_kernel<T, ST, VEC, NV, R>, grid, dim3(128), 0, stream, a);
  }
  // A head of 16 rows or fewer: one state row per lane group uses all of them.
  const dim3 grid((unsigned)(batch * a.H), (unsigned)ceil_div(a.P, 16));
  return launch_pdl(scan_update_kernel<T, ST, VEC, NV, 1>, grid, dim3(128), 0, stream, a);
}

template <typename T, typename ST>
cudaError_t launch_upd(const UpdArgs& a, i64 batch, cudaStream_t stream) {
  constexpr int V = 16 / (int)sizeof(ST);
  const bool vec = reinterpret_cast<uintptr_t>(a.state) % 16 == 0 && a.N % V == 0 && a.ss_r % V == 0 &&
                   a.ss_h % V == 0 && a.ss_p % V == 0;
  if (vec) {
    const i64 need = ceil_div(a.N, 8 * V);
    if (need <= 1) return launch_upd_n<T, ST, V, 1>(a, batch, stream);
    if (need <= 2) return launch_upd_n<T, ST, V, 2>(a, batch, stream);
    if (need <= 4) return launch_upd_n<T, ST, V, 4>(a, batch, stream);
    if constexpr (V == 4) return launch_upd_n<T, ST, V, 8>(a, batch, stream);
    return cudaErrorInvalidValue;
  }
  if (a.N <= 32) return launch_upd_n<T, ST, 1, 4>(a, batch, stream);
  if (a.N <= 128) return launch_upd_n<T, ST, 1, 16>(a, batch, stream);
  return launch_upd_n<T, ST, 1, 32>(a, batch, stream);
}

// ---- host side ----

bool dtype_known(int d) { return d == CC1D_F16 || d == CC1D_BF16 || d == CC1D_F32; }

// Makes the device that holds `ptr` current on the calling thread.
int use_device_of(const void* ptr, const char* what) {
  cudaPointerAttributes at;
  if (cudaPointerGetAttributes(&at, ptr) == cudaSuccess && at.type == cudaMemoryTypeDevice && at.device >= 0) {
    int cur = -1;
    if (cudaGetDevice(&cur) == cudaSuccess && cur != at.device) {
      const cudaError_t e = cudaSetDevice(at.device);
      if (e != cudaSuccess) return report_cuda_error(e, what);
    }
  } else {
    (void)cudaGetLastError();
  }
  return CC1D_OK;
}

int check_shapes(const char* what, int dtype, int dt_dtype, int state_dtype, i64 H, i64 P, i64 G, i64 N) {
  if (!dtype_known(dtype)) return report_error(CC1D_ERR_UNSUPPORTED, "%s: unsupported dtype code %d", what, dtype);
  if ((dt_dtype != dtype && dt_dtype != CC1D_F32) || (state_dtype != dtype && state_dtype != CC1D_F32))
    return report_error(CC1D_ERR_UNSUPPORTED, "%s: dt and states must be in the data's type or fp32", what);
  if (H < 0 || P < 0 || G < 0 || N < 0) return report_error(CC1D_ERR_INVALID_ARGUMENT, "%s: negative shape", what);
  if (H > 0 && (G < 1 || H % G != 0))
    return report_error(CC1D_ERR_INVALID_ARGUMENT, "%s: nheads (%lld) must be a multiple of ngroups (%lld)", what,
                        (long long)H, (long long)G);
  if (N > kMaxState)
    return report_error(CC1D_ERR_UNSUPPORTED, "%s: dstate must be at most %d (got %lld)", what, kMaxState, (long long)N);
  if (H > 65535 || P > 65535) return report_error(CC1D_ERR_UNSUPPORTED, "%s: nheads and headdim must fit 16 bits", what);
  return CC1D_OK;
}

struct ScanPlan {
  bool empty, tc, split;
};

// Chooses the kernel and how sequences are cut; fills everything in `a` but
// the workspace pointers.
int plan_scan(const cc1d_scan_params* p, ScanArgs* a, ScanPlan* plan) {
  if (p == nullptr) return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_scan: params is NULL");
  const int rc = check_shapes("cc1d_scan", p->dtype, p->dt_dtype, p->init_dtype, p->nheads, p->headdim, p->ngroups, p->dstate);
  if (rc != CC1D_OK) return rc;
  if (p->batch < 0 || p->seqlen < 0 || p->num_seqs < 0 || p->max_seqlen < 0)
    return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_scan: negative shape");
  if (p->cu_seqlens != nullptr && p->batch != 1)
    return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_scan: cu_seqlens needs batch == 1 (got %lld)", (long long)p->batch);
  std::memset(a, 0, sizeof(*a));
  std::memset(plan, 0, sizeof(*plan));
  const i64 nseq = p->cu_seqlens ? p->num_seqs : p->batch;
  plan->empty = p->nheads == 0 || p->headdim == 0 ||
                (nseq == 0 ? (p->batch == 0 || p->seqlen == 0 || p->cu_seqlens == nullptr)
                           : (p->seqlen == 0 && p->final_states == nullptr));
  if (plan->empty) return CC1D_OK;
  // Token counts and the launch's blocks (a segment has 64 tokens or more) fit 31 bits.
  if (p->seqlen > 0x7fffffffLL - 65536 || (nseq + (nseq > 0 ? p->seqlen / 64 : 0)) * p->nheads > 0x7fffffffLL)
    return report_error(CC1D_ERR_UNSUPPORTED, "cc1d_scan: too many sequences or tokens");
  if ((p->seqlen > 0 && (!p->x || !p->dt || !p->y || (p->dstate > 0 && (!p->B || !p->C)))) || !p->A)
    return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_scan: x, dt, A, B, C and y are required");
  *a = ScanArgs{p->x, p->x_batch_stride, p->x_seq_stride, p->x_head_stride, p->x_dim_stride,
                p->dt, p->dt_batch_stride, p->dt_seq_stride, p->dt_head_stride,
                p->B, p->B_batch_stride, p->B_seq_stride, p->B_group_stride, p->B_state_stride,
                p->C, p->C_batch_stride, p->C_seq_stride, p->C_group_stride, p->C_state_stride,
                p->A, p->D, p->dt_bias, p->cu_seqlens,
                p->initial_states, p->init_seq_stride, p->init_head_stride,
                p->y, p->y_batch_stride, p->y_seq_stride, p->y_head_stride,
                p->final_states, p->final_seq_stride, p->final_head_stride,
                nullptr, nullptr, p->seqlen, (int)p->nheads, (int)p->headdim, (int)p->dstate, (int)p->ngroups,
                (int)(p->nheads / p->ngroups), (int)nseq, 0, 1, 0, 0,
                p->dt_softplus ? 1 : 0, p->dt_dtype == CC1D_F32 ? 1 : 0,
                p->init_dtype == CC1D_F32 ? 1 : 0};
  a->seg_len = std::max<i64>(1, p->seqlen);
  a->segs = 1;
  a->items = nseq;
  if (nseq == 0 || p->seqlen == 0) return CC1D_OK;
  // The tensor cores take a block of 128 tokens' time for any part of one, the
  // walk its tokens' and its state's.  Where they meet, by measurement (tensor
  // cores | walk, us; 2560 rows of sequence and head, 16-bit data):
  //   64 x 128, 5120 rows   1 token 236 | 371, 16 tokens 238 | 419
  //   64 x 64               1 token 86 | 45, 16 tokens 88 | 70, 64 tokens 92 | 179
  //   64 x 32               16 tokens 78 | 38, 64 tokens 81 | 99
  //   16 x 64               16 tokens 73 | 29, 64 tokens 74 | 89
  // and with few rows (96 of 64 x 64, 16 tokens 10.6 | 11.3) somewhat earlier.
  const i64 mean = p->cu_seqlens ? ceil_div(p->seqlen, nseq) : p->seqlen;
  const bool enough = (a->P >= 64 && a->N > 64) || mean >= 48 || mean * a->P * a->N >= 65536;
  plan->tc = enough && scan_tc_eligible(p->dtype, *a, p->batch);
  DeviceInfo dev;
  const cudaError_t de = device_info(&dev);
  const i64 sms = de == cudaSuccess ? dev.sms : 148;
  if (de != cudaSuccess) (void)cudaGetLastError();  // sizes may be asked for without a GPU
  if (plan->tc && p->cu_seqlens == nullptr) {
    // One CTA an SM, so rows run in waves.  Rows may be cut into k segments, all
    // of them or those that fill no wave; the first pass over segments (states
    // only) takes about 0.65 of the second's time, a wave about one block more.
    const i64 rows = nseq * scan_tc_pairs(*a), blocks = ceil_div(p->seqlen, kScanBlock);
    a->whole = rows;
    double best = (double)ceil_div(rows, sms) * (blocks + 1);
    for (int all = 0; all < 2; ++all) {
      const i64 cut = all ? rows : rows % sms;
      for (i64 k = 2; cut > 0 && k <= std::min<i64>(blocks / 2, 64); ++k) {
        const i64 len = ceil_div(blocks, k);
        if (ceil_div(blocks, len) != k) continue;
        const double cost = (double)((rows - cut) / sms) * (blocks + 1) + (double)ceil_div(cut * k, sms) * (len + 1) +
                            (double)ceil_div(cut * (k - 1), sms) * (0.65 * len + 1);
        if (cost < 0.95 * best) {
          best = cost;
          plan->split = true;
          a->whole = rows - cut;
          a->seg_len = len * kScanBlock;
          a->segs = (int)k;
        }
      }
    }
    return CC1D_OK;
  }
  // The others are split when their rows alone do not fill the SMs (one CTA
  // each on the tensor cores, about four blocks of the walk), into segments of
  // two blocks or 64 tokens at least; packed ones as if they were one.
  const i64 rows = (p->cu_seqlens ? 1 : nseq) * (plan->tc ? scan_tc_pairs(*a) : a->H * ceil_div(a->P, 64));
  const i64 least = plan->tc ? 2 * kScanBlock : 64, unit = plan->tc ? kScanBlock : 16;
  const i64 segs = std::min<i64>((plan->tc ? sms : 4 * sms) / rows, p->seqlen / least);
  if (segs > 1) {
    const i64 len = ceil_div(ceil_div(p->seqlen, segs), unit) * unit;
    const i64 longest = p->cu_seqlens && p->max_seqlen == 0 ? p->seqlen : p->cu_seqlens ? p->max_seqlen : p->seqlen;
    if (longest > len) {
      plan->split = true;
      a->seg_len = len;
      a->segs = (int)ceil_div(p->seqlen, len);
      a->items = p->cu_seqlens ? nseq + p->seqlen / len : nseq * a->segs;
    }
  }
  return CC1D_OK;
}

size_t scan_workspace(const ScanArgs& a, const ScanPlan& plan) {
  if (plan.empty || !plan.split) return 0;
  return (size_t)(plan.tc ? scan_tc_parts(a) : a.items * a.H) * ((size_t)a.P * a.N + 1) * sizeof(float);
}

template <typename T>
cudaError_t launch_outside(const ScanArgs& a, cudaStream_t s) {
  return launch_pdl(scan_outside_kernel<T>, dim3(148), dim3(256), 0, s, a);
}

}  // namespace

}  // namespace cc1d

using namespace cc1d;

extern "C" int cc1d_scan_workspace_size(const cc1d_scan_params* p, size_t* bytes) {
  if (bytes == nullptr) return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_scan_workspace_size: bytes is NULL");
  ScanArgs a;
  ScanPlan plan;
  const int rc = plan_scan(p, &a, &plan);
  *bytes = rc == CC1D_OK ? scan_workspace(a, plan) : 0;
  return rc;
}

extern "C" int cc1d_scan(const cc1d_scan_params* p, void* stream) {
  ScanArgs a;
  ScanPlan plan;
  int rc = plan_scan(p, &a, &plan);
  if (rc != CC1D_OK || plan.empty) return rc;
  const size_t need = scan_workspace(a, plan);
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need))
    return report_error(CC1D_ERR_WORKSPACE, "cc1d_scan: workspace of %zu bytes required", need);
  rc = use_device_of(p->seqlen > 0 ? p->y : (const void*)p->final_states, "cc1d_scan: cudaSetDevice");
  if (rc != CC1D_OK) return rc;
  if (need > 0) {
    a.part = static_cast<float*>(p->workspace);
    a.decay = a.part + (size_t)(plan.tc ? scan_tc_parts(a) : a.items * a.H) * a.P * a.N;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (plan.tc)
    e = launch_scan_tc(p->dtype, a, p->batch, s);
  else if (a.nseq > 0)
    e = p->dtype == CC1D_F16    ? launch_walk<__half>(a, plan.split, s)
        : p->dtype == CC1D_BF16 ? launch_walk<__nv_bfloat16>(a, plan.split, s)
                                : launch_walk<float>(a, plan.split, s);
  if (e != cudaSuccess) return report_cuda_error(e, "cc1d_scan launch");
  if (a.cu != nullptr && a.L > 0) {
    e = p->dtype == CC1D_F16    ? launch_outside<__half>(a, s)
        : p->dtype == CC1D_BF16 ? launch_outside<__nv_bfloat16>(a, s)
                                : launch_outside<float>(a, s);
    if (e != cudaSuccess) return report_cuda_error(e, "cc1d_scan (tokens outside the sequences)");
  }
  return CC1D_OK;
}

extern "C" int cc1d_scan_update(const cc1d_scan_update_params* p, void* stream) {
  if (p == nullptr) return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_scan_update: params is NULL");
  int rc = check_shapes("cc1d_scan_update", p->dtype, p->dt_dtype, p->state_dtype, p->nheads, p->headdim, p->ngroups, p->dstate);
  if (rc != CC1D_OK) return rc;
  if (p->batch < 0 || p->state_rows < 0) return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_scan_update: negative shape");
  if (p->batch == 0 || p->nheads == 0 || p->headdim == 0) return CC1D_OK;
  if (p->batch * p->nheads > 0x7fffffffLL) return report_error(CC1D_ERR_UNSUPPORTED, "cc1d_scan_update: batch is too large");
  if (!p->x || !p->dt || !p->A || !p->y || (p->dstate > 0 && (!p->B || !p->C || (!p->state && p->state_rows > 0))))
    return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_scan_update: x, dt, A, B, C, state and y are required");
  if (p->state_indices == nullptr && p->state_rows < p->batch)
    return report_error(CC1D_ERR_INVALID_ARGUMENT, "cc1d_scan_update: state has %lld rows for batch %lld",
                        (long long)p->state_rows, (long long)p->batch);
  rc = use_device_of(p->y, "cc1d_scan_update: cudaSetDevice");
  if (rc != CC1D_OK) return rc;
  UpdArgs a{p->x, p->x_batch_stride, p->x_head_stride, p->x_dim_stride,
            p->dt, p->dt_batch_stride, p->dt_head_stride,
            p->B, p->B_batch_stride, p->B_group_stride, p->B_state_stride,
            p->C, p->C_batch_stride, p->C_group_stride, p->C_state_stride,
            p->A, p->D, p->dt_bias,
            p->state, p->state_row_stride, p->state_head_stride, p->state_dim_stride,
            p->state_indices, p->out_state_indices, p->y, p->y_batch_stride, p->y_head_stride,
            p->state_rows, (int)p->nheads, (int)p->headdim, (int)p->dstate, (int)(p->nheads / p->ngroups),
            p->dt_softplus ? 1 : 0, p->dt_dtype == CC1D_F32 ? 1 : 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f32 = p->state_dtype == CC1D_F32;
  cudaError_t e;
  if (p->dtype == CC1D_F16)
    e = f32 ? launch_upd<__half, float>(a, p->batch, s) : launch_upd<__half, __half>(a, p->batch, s);
  else if (p->dtype == CC1D_BF16)
    e = f32 ? launch_upd<__nv_bfloat16, float>(a, p->batch, s) : launch_upd<__nv_bfloat16, __nv_bfloat16>(a, p->batch, s);
  else
    e = launch_upd<float, float>(a, p->batch, s);
  if (e != cudaSuccess) return report_cuda_error(e, "cc1d_scan_update launch");
  return CC1D_OK;
}
