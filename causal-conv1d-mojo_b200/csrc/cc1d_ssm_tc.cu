// State space scan over prompts on the 5th-generation tensor cores
// (tcgen05, bf16 / fp16 data).
//
// Mathematics.  With a_t = dt_t A <= 0 and c_i = a_1 + ... + a_i inside a
// block of Q = 128 tokens that starts from the state S (P x N),
//   y_i  = exp(c_i) S C_i + sum_{j <= i} exp(c_i - c_j) dt_j (C_i . B_j) x_j + D x_i
//   S'   = exp(c_Q) S + sum_j exp(c_Q - c_j) dt_j x_j B_j^T
// which is four matrix products per block, all with 128 rows:
//   G     = C B^T                       (tokens x tokens, K = N)
//   inter = C S^T                       (tokens x p, K = N)
//   intra = M X, M_ij = G_ij exp(c_i - c_j) dt_j for j <= i  (K = tokens)
//   dS^T  = (w X)^T B, w_j = exp(c_Q - c_j) dt_j             (p x n, K = tokens)
// A CTA runs one sequence (or segment of it) for two heads of one group
// (one head when headdim > 64): 128 columns of x.  The heads share B, C and
// G, which halves the loads from L2 per head and the products for G.  The
// state stays in registers in fp32 from the first block to the last.
//
// Decays.  exp(c_i - c_j) is never formed from sums over the whole block,
// whose rounding would show: sums run inside sub-blocks of 32 tokens, and
// for j in an earlier sub-block than i
//   exp(c_i - c_j) = exp(sum from j+1 to the end of j's sub-block)
//                    * exp(whole sub-blocks between) * exp(sum up to i in its own),
// a value per j, times a value per i and sub-block: 32 exponentials per row
// instead of 128.  All factors are <= 1, so nothing overflows.  w_j sums from
// the block's end backwards.  A step's a_t is held at -160 in base 2 (its
// decay is 0 in fp32 from -150 on), which keeps the sums exact enough when
// single steps forget everything.
//
// Rounding.  Operands of a product are 16-bit.  x, B and C are; M and, for
// `inter`, the state are rounded once to the data's type, as y is at its end.
// w X is what the carried state is made of: where final states are asked for
// it is split into 16-bit terms and the product is taken of each, three of
// bf16 (24 bits) or two of fp16 (22 bits), so the states keep fp32 accuracy
// (one bf16 term leaves a relative error of 1.7e-3, two 3e-6).  Without final
// states one term is enough for y.  fp16 has few exponents: there w X is
// scaled by a power of two, per row p to just under fp16's largest value (or
// with one term per head to w < 1), which dS is scaled back by.
//
// Roles (20 warps, one CTA per SM):
//   warp 0       TMA: B and X in rings of two blocks, C in one buffer
//                (released as soon as G and inter have read it)
//   warp 1       allocates TMEM, issues every tcgen05.mma (one lane)
//   warp 2       step lengths and decay factors of the next block
//   warps 4-11   tokens: thread = token row.  M from G, in place in TMEM (a
//                block of 32 fp32 columns becomes 16 + 16 columns, one head
//                each); scales inter by exp(c_i), so that intra accumulates
//                onto it; y + D x over x in shared memory, then out
//   warps 12-19  state: thread = row p of S, half of n.  (w X)^T into TMEM,
//                S = exp(c_Q) S + dS, 16-bit copy to shared memory
// TMEM (512 columns): G / M 128, y 128, dS 128, (w X)^T 4 slots of 32 (64
// tokens each).  (w X)^T comes from TMEM and not from shared memory because
// the products' operands already take most of the shared-memory bandwidth.
// Order of the products of block b: first half of dS, G, inter, rest of dS,
// intra; so M is computed while dS runs, and the state is updated while
// intra runs.
//
// Every mbarrier wait is bounded; a wait that gives up sets an abort flag
// and ends its role, the others' waits then give up in turn, outstanding
// copies and products are waited for (bounded) and TMEM is released.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "cc1d.h"
#include "cc1d_dispatch.cuh"
#include "cc1d_ssm.cuh"
#include "cc1d_tma.cuh"

namespace cc1d {

namespace {

constexpr int kQ = 128;                 // tokens per block
constexpr int kThreads = 640;
constexpr unsigned kBox = kQ * 128;     // bytes of a [128 rows][64 16-bit columns] tile
constexpr unsigned kTile = 2 * kBox;
constexpr unsigned kOffB = 0;                    // 2 stages
constexpr unsigned kOffX = kOffB + 2 * kTile;    // 2 stages
constexpr unsigned kOffC = kOffX + 2 * kTile;
constexpr unsigned kOffS = kOffC + kTile;
constexpr unsigned kOffCum = kOffS + kTile;

// Decay factors of one head in one block.
struct Cum {
  float l[kQ];      // base-2 sum inside the sub-block, up to and with the token
  float d[kQ];      // step length
  float u[kQ];      // d * 2^(sum after the token inside its sub-block)
  float w[kQ];      // d * 2^(sum after the token in the block) * scale
  float e[kQ];      // 2^(sum up to and with the token in the block)
  float tot[4];     // sums of the sub-blocks
  float dec;        // 2^(sum of the block)
  float unscale;    // 1 / scale
  float pad[2];
};
constexpr unsigned kOffMax = kOffCum + 2 * 2 * sizeof(Cum);  // fp16: largest |w x| per row, [half][128]
constexpr unsigned kOffBar = kOffMax + 2 * kQ * 4;

struct Bars {
  uint64_t fullB[2], fullX[2], fullC;
  uint64_t emptyB[2], emptyX[2], emptyC;
  uint64_t cumF[2], cumE[2];
  uint64_t gR, iR, pR, yR, yF;
  uint64_t wR[4], wF[4];
  uint64_t dR, dF, sR, end;
  uint64_t ySync, xSync, mSync;  // among the token warps, among the state warps
  uint32_t tmem;
  int abort;
};
constexpr unsigned kSmem = kOffBar + sizeof(Bars) + 1024;
static_assert(kSmem <= 232448, "exceeds the shared memory a block may use");
static_assert(kOffCum % 16 == 0 && sizeof(Cum) % 16 == 0 && kOffBar % 8 == 0, "alignment");

constexpr uint32_t kColG = 0, kColY = 128, kColD = 256, kColW = 384;

struct alignas(64) TcArgs {
  CUtensorMap mx, mb, mc;
  ScanArgs a;
  int npairs, ppg;   // CTAs per segment; per group
  int nb;            // 64-column blocks of the state size
};

// ---- tcgen05 (one CTA) ----
__device__ __forceinline__ void tm_alloc(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tm_dealloc(uint32_t t) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(t) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// D (+)= A B, A and B in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// D (+)= A B, A in tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tm_ld32(uint32_t t, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t t, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31]), "r"(t)
      : "memory");
}
__device__ __forceinline__ void tm_st8(uint32_t t, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
      "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(t)
      : "memory");
}
__device__ __forceinline__ void tm_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory descriptor of a tile in the 128-byte swizzle (rows of 128
// bytes, groups of 8 rows 1024 bytes apart).  K-major operand: K runs along
// the row.  MN-major operand: K runs over rows, and `lbo` is the distance
// between 64-element column blocks.
__device__ __forceinline__ uint64_t sw_desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptor, kind::f16, M = 128, fp32 accumulator.
template <typename T>
__device__ __forceinline__ uint32_t i_desc(int n, bool b_mn) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3)
      : "memory");
}

// Bounded wait that also gives up when another role has.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, unsigned parity, volatile int* abort_flag) {
  for (unsigned i = 0; i < kSpinLimit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 255u && *abort_flag) return false;
  }
  atomicAdd(&g_cc1d_wait_timeouts, 1u);
  *abort_flag = 1;
  return false;
}

// One vote of a warp: all its lanes' accesses before are ordered before it.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// TERMS: 16-bit terms of w X.  PART: only the segment's state from zero.
// WIDE: one head of up to 128 columns instead of two of up to 64.
template <typename T, int TERMS, bool PART, bool WIDE>
__global__ void __launch_bounds__(kThreads, 1) scan_tc_kernel(const __grid_constant__ TcArgs p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Bars* bar = reinterpret_cast<Bars*>(sm + kOffBar);
  Cum(*cum)[2] = reinterpret_cast<Cum(*)[2]>(sm + kOffCum);  // [stage][head]
  volatile int* abort_flag = &bar->abort;
  const ScanArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  griddep_wait();
  ScanItem it;
  const i64 item = blockIdx.x / p.npairs;
  const int pair = blockIdx.x % p.npairs;
  if (!scan_locate(a, item, &it)) return;
  if (PART && it.seg + 1 >= it.nsegs) return;
  const int g = pair / p.ppg;
  const int h0 = g * a.R + (pair % p.ppg) * (WIDE ? 1 : 2);
  const int nh = WIDE ? 1 : min(2, (g + 1) * a.R - h0);  // heads of this CTA
  const int nblk = (int)((it.t1 - it.t0 + kQ - 1) / kQ);

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar->fullB[s], 1);
      mbar_init(&bar->fullX[s], 1);
      mbar_init(&bar->emptyB[s], 1);
      mbar_init(&bar->emptyX[s], 8);
      mbar_init(&bar->cumF[s], 1);
      mbar_init(&bar->cumE[s], PART ? 8 : 16);
    }
    mbar_init(&bar->fullC, 1);
    mbar_init(&bar->emptyC, 1);
    mbar_init(&bar->gR, 1);
    mbar_init(&bar->iR, 1);
    mbar_init(&bar->pR, 8);
    mbar_init(&bar->yR, 1);
    mbar_init(&bar->yF, 8);
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bar->wR[s], 8);
      mbar_init(&bar->wF[s], 1);
    }
    mbar_init(&bar->dR, 1);
    mbar_init(&bar->dF, 8);
    mbar_init(&bar->sR, 8);
    mbar_init(&bar->end, 1);
    mbar_init(&bar->ySync, 8);
    mbar_init(&bar->xSync, 8);
    mbar_init(&bar->mSync, 8);
    bar->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tm_alloc(&bar->tmem);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = bar->tmem;
  // A wait that gave up ends its role (for a whole warp: of all its lanes).
#define CC1D_WAIT1(b, ph)                                  \
  if (!wait_or_abort(&bar->b, (ph)&1, abort_flag)) break;
#define CC1D_WAITW(b, ph)                                                      \
  if (__any_sync(kFull, !wait_or_abort(&bar->b, (ph)&1, abort_flag))) break;

  if (warp == 0) {
    // ---------------- TMA ----------------
    if (lane == 0) {
      prefetch_tensormap(&p.mx);
      prefetch_tensormap(&p.mb);
      if (!PART) prefetch_tensormap(&p.mc);
      unsigned nB = 0, nX = 0, nC = 0;  // loads issued
      for (unsigned c = 0; c < (unsigned)nblk; ++c) {
        const unsigned s = c & 1;
        const int t = (int)(it.t0 + (i64)c * kQ), b = (int)it.batch;
        if (c >= 2) { CC1D_WAIT1(emptyB[s], (c >> 1) - 1) }
        mbar_arrive_expect_tx(&bar->fullB[s], p.nb * kBox);
        for (int k = 0; k < p.nb; ++k) tma_tile(sm + kOffB + s * kTile + k * kBox, &p.mb, &bar->fullB[s], 64 * k, g, t, b);
        ++nB;
        if (!PART) {
          if (c >= 1) { CC1D_WAIT1(emptyC, c - 1) }
          mbar_arrive_expect_tx(&bar->fullC, p.nb * kBox);
          for (int k = 0; k < p.nb; ++k) tma_tile(sm + kOffC + k * kBox, &p.mc, &bar->fullC, 64 * k, g, t, b);
          ++nC;
        }
        if (c >= 2) { CC1D_WAIT1(emptyX[s], (c >> 1) - 1) }
        mbar_arrive_expect_tx(&bar->fullX[s], kTile);
        for (int k = 0; k < 2; ++k)
          tma_tile(sm + kOffX + s * kTile + k * kBox, &p.mx, &bar->fullX[s], WIDE ? 64 * k : 0, WIDE ? h0 : h0 + k, t, b);
        ++nX;
      }
      // Nothing may land after the block has gone (normally all has landed).
      mbar_drain(bar->fullB, nB, 2);
      mbar_drain(bar->fullX, nX, 2);
      if (!PART) mbar_drain(&bar->fullC, nC, 1);
    }
  } else if (warp == 1) {
    // ---------------- matrix products ----------------
    if (lane == 0) {
      const uint32_t sB = smem_u32(sm + kOffB), sX = smem_u32(sm + kOffX), sC = smem_u32(sm + kOffC), sS = smem_u32(sm + kOffS);
      const uint32_t dG = tmem + kColG, dY = tmem + kColY, dD = tmem + kColD, dW = tmem + kColW;
      const uint32_t id_nn = i_desc<T>(128, false);             // G, inter
      const uint32_t id_in = i_desc<T>(WIDE ? 128 : 64, true);  // intra
      const uint32_t id_st = i_desc<T>(64 * p.nb, true);        // dS
      const int ksteps = 4 * p.nb;
      unsigned n = 0;  // slots of w X used
      for (unsigned c = 0; c < (unsigned)nblk; ++c) {
        const unsigned s = c & 1;
        bool ok = true;
        // dS += (term, 64 tokens) of each slot; two halves of TERMS slots.
        auto state = [&](int from, int to) {
          for (int k = from; k < to && ok; ++k, ++n) {
            const unsigned sl = n & 3;
            ok = wait_or_abort(&bar->wR[sl], (n >> 2) & 1, abort_flag);
            if (!ok) return;
            tc_after();
            const int half = k / TERMS;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma_ts(dD, dW + sl * 32 + ks * 8, sw_desc(sB + s * kTile + (half * 4 + ks) * 2048, kBox), id_st, (k | ks) != 0);
            tc_commit(&bar->wF[sl]);
          }
        };
        CC1D_WAIT1(fullB[s], c >> 1)
        if (c > 0) { CC1D_WAIT1(dF, c - 1) }
        tc_after();
        if (TERMS > 1 || PART) state(0, TERMS);
        if (!ok) break;
        if (!PART) {
          CC1D_WAIT1(fullC, c)
          // intra of the block before reads M where G goes.
          if (c > 0) { CC1D_WAIT1(yR, c - 1) }
          tc_after();
          for (int ks = 0; ks < ksteps; ++ks) {
            const uint32_t o = (ks >> 2) * kBox + (ks & 3) * 32;
            mma_ss(dG, sw_desc(sC + o, 16), sw_desc(sB + s * kTile + o, 16), id_nn, ks != 0);
          }
          tc_commit(&bar->gR);
          CC1D_WAIT1(sR, c)
          if (c > 0) { CC1D_WAIT1(yF, c - 1) }
          tc_after();
          for (int ks = 0; ks < ksteps; ++ks) {
            const uint32_t o = (ks >> 2) * kBox + (ks & 3) * 32;
            mma_ss(dY, sw_desc(sC + o, 16), sw_desc(sS + o, 16), id_nn, ks != 0);
          }
          tc_commit(&bar->iR);
          tc_commit(&bar->emptyC);
        }
        state(TERMS > 1 || PART ? TERMS : 0, 2 * TERMS);
        if (!ok) break;
        tc_commit(&bar->dR);
        tc_commit(&bar->emptyB[s]);
        if (!PART) {
          CC1D_WAIT1(pR, c)
          CC1D_WAIT1(fullX[s], c >> 1)
          tc_after();
          for (int hs = 0; hs < (WIDE ? 1 : 2); ++hs)
            for (int ks = 0; ks < 8; ++ks)
              mma_ts(dY + hs * 64, dG + 32 * (ks >> 1) + 16 * hs + 8 * (ks & 1),
                     sw_desc(sX + s * kTile + hs * kBox + ks * 2048, kBox), id_in, 1);
          tc_commit(&bar->yR);
        }
      }
      if (nblk > 0) {  // the block stays until its last products are done
        tc_commit(&bar->end);
        (void)mbar_wait(&bar->end, 0);
      }
    }
  } else if (warp == 2) {
    // ---------------- steps and decays ----------------
    float A2[2], bias[2];
    for (int k = 0; k < 2; ++k) {
      const bool ok = k < nh;
      A2[k] = ok ? a.A[h0 + k] * kLog2e : 0.f;
      bias[k] = ok && a.dt_bias ? a.dt_bias[h0 + k] : 0.f;
    }
    const i64 o = it.batch * a.ds_b + h0 * a.ds_h;
    for (unsigned c = 0; c < (unsigned)nblk; ++c) {
      const unsigned s = c & 1;
      float d[2][4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const i64 t = it.t0 + (i64)c * kQ + q * 32 + lane;
          d[k][q] = k < nh && t < it.t1 ? scan_step<T>(a, o + k * a.ds_h + t * a.ds_t, bias[k]) : 0.f;
        }
      }
      if (c >= 2) { CC1D_WAITW(cumE[s], (c >> 1) - 1) }
      for (int k = 0; k < (WIDE ? 1 : 2); ++k) {
        Cum& u = cum[s][k];
        float l[4], r[4], tot[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float v = fmaxf(d[k][q] * A2[k], -160.f);
          l[q] = v;
          r[q] = v;
#pragma unroll
          for (int sh = 1; sh < 32; sh <<= 1) {
            const float up = __shfl_up_sync(kFull, l[q], sh), dn = __shfl_down_sync(kFull, r[q], sh);
            if (lane >= sh) l[q] += up;
            if (lane + sh < 32) r[q] += dn;
          }
          tot[q] = __shfl_sync(kFull, r[q], 0);
          r[q] = __shfl_down_sync(kFull, r[q], 1);
          if (lane == 31) r[q] = 0.f;
        }
        float w[4], big = 0.f;
        float before = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float later = 0.f;
#pragma unroll
          for (int j = 3; j > q; --j) later += tot[j];
          const int t = q * 32 + lane;
          u.l[t] = l[q];
          u.d[t] = d[k][q];
          u.u[t] = d[k][q] * ex2_approx(r[q]);
          w[q] = d[k][q] * ex2_approx(r[q] + later);
          u.e[t] = ex2_approx(before + l[q]);
          before += tot[q];
          big = fmaxf(big, fabsf(w[q]));
        }
        // fp16, one term: the largest weight into [1/2, 1), so that w x cannot overflow.
        float scale = 1.f, unscale = 1.f;
        if (std::is_same<T, __half>::value && TERMS == 1) {
#pragma unroll
          for (int sh = 16; sh > 0; sh >>= 1) big = fmaxf(big, __shfl_xor_sync(kFull, big, sh));
          const int ex = min(max((int)((__float_as_uint(big) >> 23) & 255u), 27), 227);
          scale = __uint_as_float((unsigned)(253 - ex) << 23);
          unscale = __uint_as_float((unsigned)(ex + 1) << 23);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) u.w[q * 32 + lane] = w[q] * scale;
        if (lane == 0) {
#pragma unroll
          for (int q = 0; q < 4; ++q) u.tot[q] = tot[q];
          u.dec = ex2_approx(before);
          u.unscale = unscale;
        }
      }
      warp_arrive(&bar->cumF[s]);
    }
  } else if (warp >= 4 && warp < 12) {
    // ---------------- tokens ----------------
    if (!PART) {
      const int q = warp & 3, hf = (warp - 4) >> 2;
      const int row = q * 32 + lane;
      const uint32_t lanes = (uint32_t)(q * 32) << 16;
      const int hs = WIDE ? 0 : hf;  // head slot of this thread's y columns
      const int yt = threadIdx.x - 128;
      const float Dh = a.D && hs < nh ? a.D[h0 + hs] : 0.f;
      for (unsigned c = 0; c < (unsigned)nblk; ++c) {
        const unsigned s = c & 1;
        CC1D_WAITW(cumF[s], c >> 1)
        const Cum* cu = cum[s];
        CC1D_WAITW(gR, c)
        tc_after();
        // M: this thread's row, sub-blocks {0, 3} or {1, 2} of the columns
        // (which shares the causal work evenly).
#pragma unroll 1
        for (int bi = 0; bi < 2; ++bi) {
          const int b = hf == 0 ? bi * 3 : 1 + bi;
          uint32_t v[32];
          const uint32_t at = tmem + lanes + kColG + 32 * b;
          if (b > q) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0u;
          } else {
            tm_ld32(at, v);
            tm_ld_wait();
            uint32_t o[32];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if (WIDE && k == 1) {
#pragma unroll
                for (int j = 16; j < 32; ++j) o[j] = 0u;
                break;
              }
              const Cum& u = cu[k];
              if (b < q) {
                float f = u.l[row];
                for (int m = b + 1; m < q; ++m) f += u.tot[m];
                f = ex2_approx(f);
                const float2 ff = f2(f, f);
                const float4* up = reinterpret_cast<const float4*>(u.u + 32 * b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float4 w4 = up[j];
                  const float2 m0 = mul2(mul2(f2(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])), f2(w4.x, w4.y)), ff);
                  const float2 m1 = mul2(mul2(f2(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])), f2(w4.z, w4.w)), ff);
                  o[16 * k + 2 * j] = Pair<T>::pack(m0);
                  o[16 * k + 2 * j + 1] = Pair<T>::pack(m1);
                }
              } else {
                const float li = u.l[row];
                const float4* lp = reinterpret_cast<const float4*>(u.l + 32 * b);
                const float4* dp = reinterpret_cast<const float4*>(u.d + 32 * b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float4 l4 = lp[j], d4 = dp[j];
                  float m[4];
                  const float lj[4] = {l4.x, l4.y, l4.z, l4.w}, dj[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    m[e] = 4 * j + e <= lane ? __uint_as_float(v[4 * j + e]) * (ex2_approx(li - lj[e]) * dj[e]) : 0.f;
                  o[16 * k + 2 * j] = Pair<T>::pack(f2(m[0], m[1]));
                  o[16 * k + 2 * j + 1] = Pair<T>::pack(f2(m[2], m[3]));
                }
              }
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = o[j];
          }
          tm_st32(at, v);
        }
        // inter times exp(c_i), in place.
        CC1D_WAITW(iR, c)
        tc_after();
        {
          const float e = cu[hs].e[row];
#pragma unroll 1
          for (int k = 0; k < 2; ++k) {
            uint32_t v[32];
            const uint32_t at = tmem + lanes + kColY + 64 * hf + 32 * k;
            tm_ld32(at, v);
            tm_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * e);
            tm_st32(at, v);
          }
        }
        tm_st_wait();
        tc_before();
        warp_arrive(&bar->pR);
        if (lane == 0) mbar_arrive(&bar->cumE[s]);
        // y + D x, over x.
        CC1D_WAITW(yR, c)
        tc_after();
        uint4* xr = reinterpret_cast<uint4*>(sm + kOffX + s * kTile + hf * kBox + row * 128);
        const int sw = row & 7;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t v[32];
          tm_ld32(tmem + lanes + kColY + 64 * hf + 32 * k, v);
          tm_ld_wait();
          if (k == 1) {
            tc_before();
            warp_arrive(&bar->yF);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 w = xr[(4 * k + j) ^ sw];
            uint32_t* wp = &w.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 xv = Pair<T>::unpack(wp[e]);
              wp[e] = Pair<T>::pack(f2(fmaf(Dh, xv.x, __uint_as_float(v[8 * j + 2 * e])),
                                       fmaf(Dh, xv.y, __uint_as_float(v[8 * j + 2 * e + 1]))));
            }
            xr[(4 * k + j) ^ sw] = w;
          }
        }
        warp_arrive(&bar->ySync);
        CC1D_WAITW(ySync, c)
        const i64 tb = it.t0 + (i64)c * kQ;
        const int nv = (int)min((i64)kQ, it.t1 - tb);
        T* y = static_cast<T*>(a.y) + it.batch * a.ys_b + tb * a.ys_t + h0 * a.ys_h;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int e = yt + 256 * k, box = e >> 10, r = (e >> 3) & 127, un = e & 7;
          const int col = (WIDE ? 64 * box : 0) + 8 * un;
          if (r < nv && col < a.P && (WIDE || box < nh)) {
            const uint4 w = *reinterpret_cast<const uint4*>(sm + kOffX + s * kTile + box * kBox + r * 128 + ((un ^ (r & 7)) << 4));
            *reinterpret_cast<uint4*>(y + r * a.ys_t + (WIDE ? 0 : box * a.ys_h) + col) = w;
          }
        }
        fence_proxy_async_smem();
        warp_arrive(&bar->emptyX[s]);
      }
    }
  } else if (warp >= 12) {
    // ---------------- state ----------------
    const int q = warp & 3, hf = (warp - 12) >> 2;
    const int row = q * 32 + lane;                   // row of dS^T
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const int hs = WIDE ? 0 : q >> 1;
    const int pr = WIDE ? row : row & 63;            // row of the head's state
    const bool live = hs < nh && pr < a.P;
    const int st = threadIdx.x - 384;
    float S[64];
    {
      const i64 e0 = (i64)pr * a.N + 64 * hf;
#pragma unroll
      for (int j = 0; j < 64; ++j) S[j] = 0.f;
      if (!PART && live) {
        const i64 h = h0 + hs;
        if (a.init) {
          const i64 o = it.seq * a.is_s + h * a.is_h + e0;
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (64 * hf + j < a.N)
              S[j] = a.init_f32 ? static_cast<const float*>(a.init)[o + j] : Cvt<T>::f(static_cast<const T*>(a.init)[o + j]);
        }
        for (int r = 0; r < it.seg; ++r) {  // the earlier segments, in order
          const i64 slot = (it.first + r) * a.H + h;
          const float dc = ex2_approx(a.decay[slot]);
          const float* part = a.part + slot * a.P * a.N + e0;
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (64 * hf + j < a.N) S[j] = fmaf(S[j], dc, part[j]);
        }
      }
    }
    // 16-bit copy of the state for inter: row p, this thread's half of n.
    auto put = [&]() {
      uint4* sr = reinterpret_cast<uint4*>(sm + kOffS + hf * kBox + row * 128);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint4 w;
        w.x = Pair<T>::pack(f2(S[8 * j], S[8 * j + 1]));
        w.y = Pair<T>::pack(f2(S[8 * j + 2], S[8 * j + 3]));
        w.z = Pair<T>::pack(f2(S[8 * j + 4], S[8 * j + 5]));
        w.w = Pair<T>::pack(f2(S[8 * j + 6], S[8 * j + 7]));
        sr[j ^ (row & 7)] = w;
      }
      fence_proxy_async_smem();
      warp_arrive(&bar->sR);
    };
    if (!PART) put();
    unsigned n = 0;      // slots of w X used
    float total = 0.f;   // base-2 log of the segment's decay
    const int xbox = q >> 1, xc = row & 63;
    constexpr bool kRowScale = std::is_same<T, __half>::value && TERMS > 1;
    for (unsigned c = 0; c < (unsigned)nblk; ++c) {
      const unsigned s = c & 1;
      CC1D_WAITW(fullX[s], c >> 1)
      CC1D_WAITW(fullB[s], c >> 1)
      unsigned char* xt = sm + kOffX + s * kTile;
      const i64 tb = it.t0 + (i64)c * kQ;
      if (a.cu != nullptr && it.t1 - tb < kQ) {
        // The rows behind the sequence's end belong to others, whatever they
        // hold: zeros keep it out of the sums.
        const int nv = (int)(it.t1 - tb);
        for (int e = nv * 8 + st; e < kQ * 8; e += 256) {
          const uint4 z = make_uint4(0u, 0u, 0u, 0u);
          reinterpret_cast<uint4*>(xt)[e] = z;
          reinterpret_cast<uint4*>(xt + kBox)[e] = z;
          for (int k = 0; k < p.nb; ++k) reinterpret_cast<uint4*>(sm + kOffB + s * kTile + k * kBox)[e] = z;
        }
        fence_proxy_async_smem();
        warp_arrive(&bar->xSync);
        CC1D_WAITW(xSync, 0)  // a sequence has one such block, its last
      }
      CC1D_WAITW(cumF[s], c >> 1)
      const Cum& u = cum[s][hs];
      // x of token t in this thread's column.
      auto x_at = [&](int t) {
        return Cvt<T>::f(*reinterpret_cast<const T*>(xt + xbox * kBox + t * 128 + ((((xc >> 3) ^ (t & 7)) << 4) | ((xc & 7) << 1))));
      };
      float scale = 1.f, unscale = u.unscale;
      if (kRowScale) {
        float m = 0.f;
#pragma unroll 8
        for (int k = 0; k < 64; ++k) {
          const int t = 64 * (k >> 5) + 32 * hf + (k & 31);
          m = fmaxf(m, fabsf(u.w[t] * x_at(t)));
        }
        float* rm = reinterpret_cast<float*>(sm + kOffMax);
        rm[hf * kQ + row] = m;
        warp_arrive(&bar->mSync);
        CC1D_WAITW(mSync, c)
        const unsigned ex = max((__float_as_uint(fmaxf(rm[row], rm[kQ + row])) >> 23) & 255u, 15u);
        scale = __uint_as_float((268u - ex) << 23);  // the largest into [2^14, 2^15)
        unscale = __uint_as_float((ex - 14u) << 23);
      }
      bool ok = true;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int k = 0; k < TERMS; ++k)
          if (n + k >= 4) ok = ok && wait_or_abort(&bar->wF[(n + k) & 3], (((n + k) >> 2) - 1) & 1, abort_flag);
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        tc_after();
        // This thread: tokens [64 half + 32 hf, + 32) of column p.
#pragma unroll
        for (int k16 = 0; k16 < 2; ++k16) {
          const int t0 = 64 * half + 32 * hf + 16 * k16;
          uint32_t o[TERMS][8];
          const float4* wp = reinterpret_cast<const float4*>(u.w + t0);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 w4 = wp[j];
            const float wj[4] = {w4.x, w4.y, w4.z, w4.w};
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[e] = wj[e] * x_at(t0 + 4 * j + e);
              if (kRowScale) v[e] *= scale;
            }
#pragma unroll
            for (int k = 0; k < TERMS; ++k) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t w = Pair<T>::pack(f2(v[2 * e], v[2 * e + 1]));
                o[k][2 * j + e] = w;
                if (k + 1 < TERMS) {
                  const float2 back = Pair<T>::unpack(w);
                  v[2 * e] -= back.x;
                  v[2 * e + 1] -= back.y;
                }
              }
            }
          }
#pragma unroll
          for (int k = 0; k < TERMS; ++k) tm_st8(tmem + lanes + kColW + ((n + k) & 3) * 32 + 16 * hf + 8 * k16, o[k]);
        }
        tm_st_wait();
        tc_before();
        __syncwarp();
        if (lane == 0) {
          for (int k = 0; k < TERMS; ++k) mbar_arrive(&bar->wR[(n + k) & 3]);
        }
        n += TERMS;
      }
      if (!ok) break;
      if (PART) warp_arrive(&bar->emptyX[s]);
      const float dec = u.dec;
      if (PART) total += u.tot[0] + u.tot[1] + u.tot[2] + u.tot[3];
      warp_arrive(&bar->cumE[s]);
      CC1D_WAITW(dR, c)
      tc_after();
      if (hf < p.nb) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t v[32];
          tm_ld32(tmem + lanes + kColD + 64 * hf + 32 * k, v);
          tm_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) S[32 * k + j] = fmaf(S[32 * k + j], dec, __uint_as_float(v[j]) * unscale);
        }
      }
      tc_before();
      warp_arrive(&bar->dF);
      if (!PART && c + 1 < (unsigned)nblk) {
        CC1D_WAITW(iR, c)  // inter has read the copy before
        put();
      }
    }
    float* out = nullptr;
    if (live) {
      const i64 h = h0 + hs;
      if (PART) {
        const i64 slot = item * a.H + h;
        out = a.part + slot * a.P * a.N;
        if (pr == 0 && hf == 0) a.decay[slot] = total;
      } else if (a.fin && it.seg + 1 == it.nsegs) {
        out = a.fin + it.seq * a.fs_s + h * a.fs_h;
      }
    }
    if (out != nullptr) {
      out += (i64)pr * a.N + 64 * hf;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (64 * hf + 4 * j < a.N)
          *reinterpret_cast<float4*>(out + 4 * j) = make_float4(S[4 * j], S[4 * j + 1], S[4 * j + 2], S[4 * j + 3]);
    }
  }
#undef CC1D_WAIT1
#undef CC1D_WAITW
  __syncwarp();
  tc_before();
  __syncthreads();
  if (warp == 1) {
    tc_after();
    tm_dealloc(tmem);
  }
}

// ---- host side ----

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static std::atomic<void*> fn{nullptr};
  void* f = fn.load(std::memory_order_acquire);
  if (f == nullptr) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess || f == nullptr)
      return nullptr;
    fn.store(f, std::memory_order_release);
  }
  return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
}

// Map over (columns, heads or groups, tokens, batch) with a [128 tokens][64
// columns] box in the 128-byte swizzle; zeros outside.
bool make_map(CUtensorMap* m, bool bf16, const void* base, i64 cols, i64 heads, i64 tokens, i64 batch, i64 s_h, i64 s_t, i64 s_b) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)cols, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)batch};
  // The stride of an axis of one element is never used, but must be valid.
  const cuuint64_t strides[3] = {(cuuint64_t)(heads > 1 ? s_h : 8) * 2, (cuuint64_t)(tokens > 1 ? s_t : 8) * 2,
                                 (cuuint64_t)(batch > 1 ? s_b : 8) * 2};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)kQ, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) set_error_detail("cuTensorMapEncodeTiled returned %d", (int)r);
  return r == CUDA_SUCCESS;
}

template <typename T, int TERMS, bool PART, bool WIDE>
cudaError_t launch_one(const TcArgs& t, cudaStream_t s) {
  static std::atomic<uint64_t> attr_done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev >= 0 && dev < 64 ? (1ull << dev) : 0ull;
  if (bit == 0 || !(attr_done.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(scan_tc_kernel<T, TERMS, PART, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
    if (e != cudaSuccess) return e;
    attr_done.fetch_or(bit, std::memory_order_acq_rel);
  }
  return launch_pdl(scan_tc_kernel<T, TERMS, PART, WIDE>, dim3((unsigned)(t.a.items * t.npairs)), dim3(kThreads), kSmem, s, t);
}

template <typename T, bool WIDE>
cudaError_t launch_all(const TcArgs& t, cudaStream_t s) {
  constexpr int kTerms = std::is_same<T, __half>::value ? 2 : 3;
  const bool exact = t.a.fin != nullptr;
  if (t.a.part != nullptr) {
    const cudaError_t e = exact ? launch_one<T, kTerms, true, WIDE>(t, s) : launch_one<T, 1, true, WIDE>(t, s);
    if (e != cudaSuccess) return e;
  }
  return exact ? launch_one<T, kTerms, false, WIDE>(t, s) : launch_one<T, 1, false, WIDE>(t, s);
}

// Strides in elements of a TMA-readable tensor: multiples of 16 bytes (of
// axes longer than 1; a broadcast axis, stride 0, is left to the other kernel).
bool stride_ok(i64 n, i64 s) { return n <= 1 || (s > 0 && s % 8 == 0 && s < ((i64)1 << 38)); }

bool tile_ok(const void* base, i64 unit, i64 heads, i64 s_h, i64 tokens, i64 s_t, i64 batch, i64 s_b) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && unit == 1 && stride_ok(heads, s_h) && stride_ok(tokens, s_t) &&
         stride_ok(batch, s_b);
}

}  // namespace

int scan_tc_pairs(const ScanArgs& a) { return a.P > 64 ? a.H : a.G * (int)ceil_div(a.R, 2); }

bool scan_tc_eligible(int dtype, const ScanArgs& a, i64 batch) {
  if (dtype == 2 || a.P < 8 || a.P > 128 || a.P % 8 || a.N < 8 || a.N > 128 || a.N % 8) return false;
  return tile_ok(a.x, a.xs_p, a.H, a.xs_h, a.L, a.xs_t, batch, a.xs_b) &&
         tile_ok(a.B, a.bs_n, a.G, a.bs_g, a.L, a.bs_t, batch, a.bs_b) &&
         tile_ok(a.C, a.cs_n, a.G, a.cs_g, a.L, a.cs_t, batch, a.cs_b) &&
         tile_ok(a.y, 1, a.H, a.ys_h, a.L, a.ys_t, batch, a.ys_b) &&
         (a.fin == nullptr || (reinterpret_cast<uintptr_t>(a.fin) % 16 == 0 && a.fs_s % 4 == 0 && a.fs_h % 4 == 0));
}

cudaError_t launch_scan_tc(int dtype, const ScanArgs& a, i64 batch, cudaStream_t stream) {
  TcArgs t;
  std::memset(&t, 0, sizeof(t));
  t.a = a;
  const bool wide = a.P > 64, bf = dtype == 1;
  t.npairs = scan_tc_pairs(a);
  t.ppg = wide ? a.R : (int)ceil_div(a.R, 2);
  t.nb = (int)ceil_div(a.N, 64);
  if (!make_map(&t.mx, bf, a.x, a.P, a.H, a.L, batch, a.xs_h, a.xs_t, a.xs_b) ||
      !make_map(&t.mb, bf, a.B, a.N, a.G, a.L, batch, a.bs_g, a.bs_t, a.bs_b) ||
      !make_map(&t.mc, bf, a.C, a.N, a.G, a.L, batch, a.cs_g, a.cs_t, a.cs_b))
    return cudaErrorInvalidValue;
  if (bf) return wide ? launch_all<__nv_bfloat16, true>(t, stream) : launch_all<__nv_bfloat16, false>(t, stream);
  return wide ? launch_all<__half, true>(t, stream) : launch_all<__half, false>(t, stream);
}

cudaError_t read_scan_wait_timeouts(unsigned* count) { return tu_read_wait_timeouts(count); }

}  // namespace cc1d
