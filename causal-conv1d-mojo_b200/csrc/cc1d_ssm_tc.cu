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
// instead of 128.  All factors are <= 1, so nothing overflows.  w_j is such a
// value per j, summed from the sub-block's end backwards, times one per
// sub-block.  A step's a_t is held at -160 in base 2 (its
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
// scaled by a power of two, per row p to just under fp16's largest value, which
// dS is scaled back by.
//
// Roles (20 warps, one CTA per SM):
//   warp 0       TMA: B and X in rings of two blocks, C in one buffer
//                (released as soon as G and inter have read it); y out
//   warp 1       allocates TMEM, issues G, inter and intra (one lane)
//   warp 2       issues dS: the chains of y and of the state meet only where
//                one needs the other, and one issuer for both would make each
//                wait for the other's barriers
//   warps 4-11   tokens: thread = token row.  Steps, decays and (bf16) the first
//                unit of (w X)^T of the next block;  M from G, in place in
//                TMEM (16 fp32 columns become 8 + 8 of pairs, one head each);
//                scales inter by exp(c_i), so that intra accumulates onto it;
//                y + D x over x in shared memory
//   warps 12-19  state: thread = row p of S, half of n.  (w X)^T into TMEM,
//                S = exp(c_Q) S + dS, 16-bit copy to shared memory
// TMEM (512 columns): G / M 128, y 128, dS 128, (w X)^T two buffers of one
// unit (32 tokens, 16 columns a term).  (w X)^T comes from TMEM and not from
// shared memory because the products' operands already take most of the
// shared-memory bandwidth.
// What a role does between two waits is kept short: with few warps it runs at
// the latency of its instructions.
//
// Measured: 8 x 2048 tokens of 80 heads of 64 x 128, bf16 with final states,
// 182 us (2.0 TB/s of data; the token-by-token walk takes 2999); one prompt
// of 16384, cut into segments, 291; 65536 packed fp16 tokens of 60 heads 556.
// Bound by the instructions of the 16 warps that feed the products, not by
// these or by memory: issue slots 53-61 % busy, the tensor pipe 35-39 %, DRAM under
// a third.
//
// A barrier tells only two phases apart: a waiter has to know that the phase
// before the one it waits for is over, and the one after must not end before
// it has looked.  So a waiter waits for every phase of a barrier in turn, and
// barriers are kept per stage, or per unit of a block, where the other side
// could be a block ahead.
//
// Every mbarrier wait is bounded; after one that gave up no wait waits, the
// roles run to their ends, outstanding copies and products are waited for
// (bounded), TMEM is released and the launch is counted in
// cc1d_device_status.
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

// Steps and decays of one head in one block.
struct Cum {
  float l[kQ];      // base-2 sum inside the sub-block, up to and with the token
  float d[kQ];      // step length
  float u[kQ];      // d * 2^(sum after the token inside its sub-block)
  float tot[4];     // sums of the sub-blocks
};
constexpr unsigned kOffMax = kOffCum + 2 * 2 * sizeof(Cum);  // fp16: largest |w x| per row, [half][128]
constexpr unsigned kOffBar = kOffMax + 2 * kQ * 4;

struct Bars {
  uint64_t fullB[2], fullX[2], fullC;
  uint64_t emptyB[2], emptyC;
  uint64_t cumF[2];
  uint64_t gR, iR, pR, yR, yF;
  uint64_t wR[4], wF[4];  // of the units of a block
  uint64_t dR, dF, sR, end, endS;
  uint64_t xF[2], yS[2];  // the state's warps have read x and the steps; y is in x's place
  uint64_t xSync, mSync;  // among the state warps
  uint32_t tmem;
  int abort;
};
constexpr unsigned kSmem = kOffBar + sizeof(Bars) + 1024;
static_assert(kSmem <= 232448, "exceeds the shared memory a block may use");
static_assert(kOffCum % 16 == 0 && sizeof(Cum) % 16 == 0 && kOffBar % 8 == 0, "alignment");

constexpr uint32_t kColG = 0, kColY = 128, kColD = 256, kColW = 384;

struct alignas(64) TcArgs {
  CUtensorMap mx, mb, mc, my;
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
__device__ __forceinline__ void tm_ld16(uint32_t t, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t t, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(t)
      : "memory");
}
__device__ __forceinline__ void tm_st8(uint32_t t, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
      "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(t)
      : "memory");
}
// Four 8x8 tiles of pairs (rows x 4 columns) into 16 lanes x 8 columns: lane
// l's registers are row l / 4 and l / 4 + 8 of column l % 4, then of l % 4 + 4.
__device__ __forceinline__ void tm_st_16x128(uint32_t t, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};" ::"r"(t), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_t(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(addr)
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

// Bounded wait by a warp (or one lane).  One that gives up sets the abort
// flag, and with the flag set no wait waits: every role then runs to its end
// on whatever is there, within its buffers, and the kernel is over.  (The
// copies stop at once: a load's barrier must not be armed a second time
// before it has completed.)
__device__ __forceinline__ void wait_for(uint64_t* bar, unsigned parity, int* abort_flag) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .u32 n, f;\n\t"
      "mov.u32 n, %2;\n\t"
      "W%=: mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1;\n\t"
      "@p bra D%=;\n\t"
      "ld.volatile.shared.u32 f, [%3];\n\t"
      "setp.ne.u32 p, f, 0;\n\t@p bra D%=;\n\t"
      "sub.u32 n, n, 1;\n\tsetp.ne.u32 p, n, 0;\n\t@p bra W%=;\n\t"
      "st.volatile.shared.u32 [%3], 1;\n\t"
      "D%=:\n\t}" ::"r"(smem_u32(bar)),
      "r"(parity), "n"(kSpinLimit), "r"(smem_u32(abort_flag))
      : "memory");
}

__device__ __forceinline__ void tma_store(const CUtensorMap* map, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

// One vote of a warp: all its lanes' accesses before are ordered before it.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.eq.u32 p, %1, 0;\n\t"
      "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(threadIdx.x & 31)
      : "memory");
}

// fp16: w X is scaled per row of dS.
template <typename T>
constexpr bool kRowScale = std::is_same<T, __half>::value;

// Takes the leading 16-bit term off two values.  bf16 terms of a split are
// cut, not rounded: the upper halves of the words, eight bits each, so that
// three of them are the 24 bits of the value.
template <typename T, bool SPLIT>
__device__ __forceinline__ uint32_t take_term(float2& v) {
  if constexpr (!SPLIT) {
    return Pair<T>::pack(v);
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t a = __float_as_uint(v.x), b = __float_as_uint(v.y);
    v = add2(v, f2(__uint_as_float((a & 0xffff0000u) ^ 0x80000000u), __uint_as_float((b & 0xffff0000u) ^ 0x80000000u)));
    return __byte_perm(a, b, 0x7632);
  } else {
    const uint32_t w = Pair<T>::pack(v);
    const float2 back = Pair<T>::unpack(w);
    v = add2(v, f2(-back.x, -back.y));
    return w;
  }
}

// w X in units of 32 tokens.  x comes transposed out of shared memory
// (ldmatrix), as lane l's columns p = l / 4 (+ 8, 16, 24) and tokens
// 2 (l % 4), + 1 of eight; the 16x128b stores put that into TMEM as rows p
// and columns of token pairs.  Of a unit a warp does 32 rows and 16 tokens:
// matrices of 8 tokens by 8 columns in the order (first 8 tokens, second 8) x
// (8 columns, next 8).
template <typename T, int TERMS>
struct Units {
  uint32_t row, col0, col1;
  int token, hf;

  __device__ __forceinline__ Units(unsigned char* sm, int q, int half, int lane) {
    row = smem_u32(sm) + kOffX + (q >> 1) * kBox + (16 * half + ((lane >> 4) << 3) + (lane & 7)) * 128;
    col0 = (((q & 1) * 4 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4;
    col1 = col0 ^ (2 << 4);
    token = 16 * half + 2 * (lane & 3);  // this lane's first token of a unit
    hf = half;
  }
  __device__ __forceinline__ void load(unsigned s, unsigned un, uint32_t (&x)[8]) const {
    const uint32_t at = row + s * kTile + un * (32 * 128);
    ldmatrix_t(at + col0, x[0], x[1], x[2], x[3]);
    ldmatrix_t(at + col1, x[4], x[5], x[6], x[7]);
  }
  // Unit n (of block n / 4, whose x is in stage s): u x g x, in terms, where
  // dS's products read it, when they have read unit n - 2 there.
  __device__ __forceinline__ void make(Bars* bar, uint32_t tm, unsigned s, unsigned n, const float* u, float g,
                                       const float (&scale)[4]) const {
    const unsigned un = n & 3;
    uint32_t x[8];
    load(s, un, x);
    const float2 w0 = mul2(*reinterpret_cast<const float2*>(u + token + 32 * un), f2(g, g));
    const float2 w1 = mul2(*reinterpret_cast<const float2*>(u + token + 32 * un + 8), f2(g, g));
    if (n >= 2) wait_for(&bar->wF[(n - 2) & 3], ((n - 2) >> 2) & 1, &bar->abort);
    tc_after();
    uint32_t o[TERMS][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float2 v = mul2((i & 2) ? w1 : w0, Pair<T>::unpack(x[i]));
      if (kRowScale<T>) v = mul2(v, f2(scale[2 * (i >> 2) + (i & 1)], scale[2 * (i >> 2) + (i & 1)]));
#pragma unroll
      for (int k = 0; k < TERMS; ++k) o[k][i] = take_term<T, (TERMS > 1)>(v);
    }
    const uint32_t at = tm + kColW + (n & 1) * (16 * TERMS) + 8 * hf;
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
      tm_st_16x128(at + 16 * k, o[k][0], o[k][1], o[k][2], o[k][3]);
      tm_st_16x128(at + 16 * k + (16u << 16), o[k][4], o[k][5], o[k][6], o[k][7]);
    }
    tm_st_wait();
    tc_before();
    warp_arrive(&bar->wR[un]);
  }
};

// TERMS: 16-bit terms of w X.  PART: only the segment's state from zero.
// WIDE: one head of up to 128 columns instead of two of up to 64.
template <typename T, int TERMS, bool PART, bool WIDE>
__global__ void __launch_bounds__(kThreads, 1) scan_tc_kernel(const __grid_constant__ TcArgs p) {
  extern __shared__ unsigned char smem_raw[];
  // An offset, not a rounded pointer, so that accesses stay shared-memory ones.
  unsigned char* sm = smem_raw + (-smem_u32(smem_raw) & 1023u);
  Bars* bar = reinterpret_cast<Bars*>(sm + kOffBar);
  Cum(*cum)[2] = reinterpret_cast<Cum(*)[2]>(sm + kOffCum);  // [stage][head]
  const ScanArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // With partial states to compute, that launch comes first and lets this one
  // start at once: its own wait is behind it by then, so what rows that are not
  // cut read is there, and only segments wait for the partial states.
  if (PART || a.part == nullptr || a.cu != nullptr || blockIdx.x >= a.whole) griddep_wait();
  if (PART) griddep_launch_dependents();
  ScanItem it;
  int pair;
  i64 part0;  // slot of segment 0 of this row's partial states; segment r is r * part_step behind
  int part_step;
  if (a.cu == nullptr) {
    // The first `whole` rows (sequence, heads) run uncut, the others in segments.
    const i64 x = (i64)blockIdx.x + (PART ? a.whole : 0), y = x - a.whole;
    const i64 row = y < 0 ? x : a.whole + y / a.segs;
    it.seq = (int)(row / p.npairs);
    pair = (int)(row - (i64)it.seq * p.npairs);
    it.nsegs = y < 0 ? 1 : a.segs;
    it.seg = y < 0 ? 0 : (int)(y % a.segs);
    it.batch = it.seq;
    it.t0 = it.seg * a.seg_len;
    it.t1 = y < 0 ? a.L : min(a.L, it.t0 + a.seg_len);
    part0 = y - it.seg;
    part_step = 1;
  } else {
    const i64 item = blockIdx.x / p.npairs;
    pair = blockIdx.x % p.npairs;
    if (!scan_locate(a, item, &it)) return;
    part0 = it.first * p.npairs + pair;
    part_step = p.npairs;
  }
  if (PART && it.seg + 1 >= it.nsegs) return;
  const int g = pair / p.ppg;
  const int h0 = g * a.R + (pair % p.ppg) * (WIDE ? 1 : 2);
  const int nh = WIDE ? 1 : min(2, (g + 1) * a.R - h0);  // heads of this CTA
  const int nblk = (int)((it.t1 - it.t0 + kQ - 1) / kQ);

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar->fullB[s], 1);
      mbar_init(&bar->fullX[s], 1);
      mbar_init(&bar->emptyB[s], PART ? 1 : 2);  // both issuers
      mbar_init(&bar->cumF[s], 8);
      mbar_init(&bar->xF[s], 8);
      mbar_init(&bar->yS[s], 8);
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
    mbar_init(&bar->endS, 1);
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
  // The first unit of a block's w X is the tokens' warps' work, which else
  // wait more than the state's.  (fp16: the row scale is of the whole block
  // and would have to come first, so the state's warps do all.)
  constexpr bool kShare = !kRowScale<T>;
  auto wait = [&](uint64_t& b, unsigned phase) { wait_for(&b, phase & 1, &bar->abort); };

  // Registers: 96 a thread at launch (61440 in all); the other warps take over
  // what the first four do not need (4 * 32 * 48 + 8 * 32 * 104 + 8 * 32 * 112
  // = 61440).
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
  if (warp == 0) {
    // ---------------- TMA ----------------
    if (lane == 0) {
      prefetch_tensormap(&p.mx);
      prefetch_tensormap(&p.mb);
      if (!PART) {
        prefetch_tensormap(&p.mc);
        prefetch_tensormap(&p.my);
      }
      const int b = (int)it.batch;
      const int np = WIDE ? 2 : nh;  // boxes of y
      // y of block c, out of x's buffer, which is free afterwards.  A block
      // that its sequence fills in part is stored by the tokens' warps.
      auto store = [&](unsigned c) {
        const unsigned s = c & 1;
        const i64 t = it.t0 + (i64)c * kQ;
        wait(bar->yS[s], c >> 1);
        if (a.cu != nullptr && it.t1 - t < kQ) return;
#pragma unroll 1
        for (int k = 0; k < np; ++k)
          tma_store(&p.my, sm + kOffX + s * kTile + k * kBox, WIDE ? 64 * k : 0, WIDE ? h0 : h0 + k, (int)t, b);
        asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
      };
      int t = (int)it.t0;
      unsigned nB = 0, nX = 0, nC = 0;  // loads issued
      volatile int* abort_flag = &bar->abort;
#pragma unroll 1
      for (unsigned c = 0; c < (unsigned)nblk; ++c, t += kQ) {
        const unsigned s = c & 1;
        if (c >= 2) wait(bar->emptyB[s], (c >> 1) - 1);
        if (*abort_flag) break;
        mbar_arrive_expect_tx(&bar->fullB[s], p.nb * kBox);
#pragma unroll 1
        for (int k = 0; k < p.nb; ++k) tma_tile(sm + kOffB + s * kTile + k * kBox, &p.mb, &bar->fullB[s], 64 * k, g, t, b);
        ++nB;
        if (c >= 2) {
          if (PART)
            wait(bar->xF[s], (c >> 1) - 1);
          else
            store(c - 2);
        }
        if (*abort_flag) break;
        mbar_arrive_expect_tx(&bar->fullX[s], kTile);
#pragma unroll 1
        for (int k = 0; k < 2; ++k)
          tma_tile(sm + kOffX + s * kTile + k * kBox, &p.mx, &bar->fullX[s], WIDE ? 64 * k : 0, WIDE ? h0 : h0 + k, t, b);
        ++nX;
        if (!PART) {
          if (c >= 1) wait(bar->emptyC, c - 1);
          if (*abort_flag) break;
          mbar_arrive_expect_tx(&bar->fullC, p.nb * kBox);
#pragma unroll 1
          for (int k = 0; k < p.nb; ++k) tma_tile(sm + kOffC + k * kBox, &p.mc, &bar->fullC, 64 * k, g, t, b);
          ++nC;
        }
      }
      if (!PART) {
        if (nblk > 1) store(nblk - 2);
        if (nblk > 0) store(nblk - 1);
      }
      // Nothing may land after the CTA has gone (normally all has landed).
      mbar_drain(bar->fullB, nB, 2);
      mbar_drain(bar->fullX, nX, 2);
      if (!PART) mbar_drain(&bar->fullC, nC, 1);
    }
  } else if (warp == 1) {
    // ---------------- products of y: G, inter, intra ----------------
    // A whole warp walks the loop, so that descriptors are uniform; one lane
    // issues.
    if (!PART) {
      const bool lead = lane == 0;
      const uint32_t sm0 = smem_u32(sm);
      const uint32_t dG = tmem + kColG, dY = tmem + kColY;
      const uint32_t id_nn = i_desc<T>(128, false);             // G, inter
      const uint32_t id_in = i_desc<T>(WIDE ? 128 : 64, true);  // intra
      const uint64_t kC = sw_desc(sm0 + kOffC, 16), kB = sw_desc(sm0 + kOffB, 16), kS = sw_desc(sm0 + kOffS, 16);
      const uint64_t mX = sw_desc(sm0 + kOffX, kBox);
      // D = C (K-major rows of Q) with a K-major B operand, K = the state size.
      auto by_state = [&](uint32_t d, uint64_t b) {
        uint64_t ca = kC;
#pragma unroll 1
        for (int k = 0; k < 2 * p.nb; ++k) {
          if (lead) {
            mma_ss(d, ca, b, id_nn, k != 0);
            mma_ss(d, ca + 2, b + 2, id_nn, 1);
          }
          // 32 bytes a step; the next 64 columns are in the next box.
          const uint32_t o = k == 1 ? (kBox - 64) >> 4 : 4;
          ca += o;
          b += o;
        }
      };
#pragma unroll 1
      for (unsigned c = 0; c < (unsigned)nblk; ++c) {
        const unsigned s = c & 1;
        wait(bar->fullB[s], c >> 1);
        wait(bar->fullC, c);
        if (c > 0) wait(bar->yR, c - 1);  // intra of the block before reads M where G goes
        tc_after();
        by_state(dG, kB + ((s * kTile) >> 4));
        if (lead) {
          tc_commit(&bar->gR);
          tc_commit(&bar->emptyB[s]);
        }
        wait(bar->sR, c);
        if (c > 0) wait(bar->yF, c - 1);
        tc_after();
        by_state(dY, kS);
        if (lead) {
          tc_commit(&bar->iR);
          tc_commit(&bar->emptyC);
        }
        wait(bar->fullX[s], c >> 1);
        if (a.cu != nullptr && it.t1 - it.t0 - (i64)c * kQ < kQ) wait(bar->xSync, 0);  // foreign rows are zeros
        wait(bar->pR, c);
        tc_after();
        // Head slot k >> 2, tokens [32 (k & 3), + 32).
        uint64_t b = mX + ((s * kTile) >> 4);
#pragma unroll 1
        for (int k = 0; k < (WIDE ? 4 : 8); ++k, b += 4096u >> 4) {
          if (lead) {
            const uint32_t m = dG + 32 * (k & 3) + 8 * (k >> 2);
            mma_ts(dY + 64 * (k >> 2), m, b, id_in, 1);
            mma_ts(dY + 64 * (k >> 2), m + 16, b + (2048u >> 4), id_in, 1);
          }
        }
        if (lead) tc_commit(&bar->yR);
      }
      if (nblk > 0) {  // the CTA stays until its last products are done
        if (lead) tc_commit(&bar->end);
        wait(bar->end, 0);
      }
    }
  } else if (warp == 2) {
    // ---------------- products of the state: dS ----------------
    const bool lead = lane == 0;
    const uint32_t dD = tmem + kColD, dW = tmem + kColW;
    const uint32_t id_st = i_desc<T>(64 * p.nb, true);
    const uint64_t mB = sw_desc(smem_u32(sm) + kOffB, kBox);
#pragma unroll 1
    for (unsigned c = 0; c < (unsigned)nblk; ++c) {
      const unsigned s = c & 1;
      wait(bar->fullB[s], c >> 1);
      if (c > 0) wait(bar->dF, c - 1);
      // Units of 32 tokens, TERMS terms each.
#pragma unroll 1
      for (unsigned u = 0; u < 4; ++u) {
        const unsigned n = 4 * c + u;
        wait(bar->wR[u], c);
        tc_after();
        const uint64_t b = mB + ((s * kTile + u * 4096u) >> 4);
        uint32_t w = dW + (n & 1) * (16 * TERMS);
#pragma unroll 1
        for (int k = 0; k < TERMS; ++k, w += 16) {
          if (lead) {
            mma_ts(dD, w, b, id_st, (k | u) != 0);
            mma_ts(dD, w + 8, b + (2048u >> 4), id_st, 1);
          }
        }
        if (lead) tc_commit(&bar->wF[u]);
      }
      if (lead) {
        tc_commit(&bar->dR);
        tc_commit(&bar->emptyB[s]);
      }
    }
    if (nblk > 0) {
      if (lead) tc_commit(&bar->endS);
      wait(bar->endS, 0);
    }
  }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---------------- tokens ----------------
    const int q = warp & 3, hf = (warp - 4) >> 2;
    const int row = q * 32 + lane;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const int hs = WIDE ? 0 : hf;  // head slot of this thread's y columns
    const int yt = threadIdx.x - 128;
    const float Dh = a.D && hs < nh ? a.D[h0 + hs] : 0.f;
    // Steps and decays: a warp takes a sub-block of a head, a lane a token.
    const bool cums = !WIDE || hf == 0;
    const bool head = cums && hf < nh;
    const float A2 = head ? a.A[h0 + hf] * kLog2e : 0.f, bias = head && a.dt_bias ? a.dt_bias[h0 + hf] : 0.f;
    i64 dto = it.batch * a.ds_b + (h0 + hf) * a.ds_h + (it.t0 + row) * a.ds_t;
    // dt of block c, asked for a block ahead and left as it is stored (a
    // conversion here would wait for it); 0 where there is none.
    auto raw_step = [&](unsigned c) {
      uint32_t d = 0u;
      if (head && it.t0 + (i64)c * kQ + row < it.t1)
        d = a.dt_f32 ? static_cast<const uint32_t*>(a.dt)[dto] : static_cast<const uint16_t*>(a.dt)[dto];
      dto += kQ * a.ds_t;
      return d;
    };
    uint32_t raw = raw_step(0);
    const Units<T, TERMS> units(sm, q, hf, lane);
    auto steps = [&](unsigned c) {
      if (cums) {
        Cum& u = cum[c & 1][hf];
        // Tokens behind the end, and a head that is not there: steps of length 0.
        float d = (a.dt_f32 ? __uint_as_float(raw) : Pair<T>::unpack(raw).x) + bias;
        d = !head || it.t0 + (i64)c * kQ + row >= it.t1 ? 0.f : a.softplus ? softplus_f(d) : d;
        if (c + 1 < (unsigned)nblk) raw = raw_step(c + 1);
        float l = fmaxf(d * A2, -160.f), r = l;
#pragma unroll
        for (int sh = 1; sh < 32; sh <<= 1) {
          const float up = __shfl_up_sync(kFull, l, sh), dn = __shfl_down_sync(kFull, r, sh);
          if (lane >= sh) l += up;
          if (lane + sh < 32) r += dn;
        }
        if (lane == 0) u.tot[q] = r;
        r = __shfl_down_sync(kFull, r, 1);
        u.l[row] = l;
        u.d[row] = d;
        u.u[row] = lane == 31 ? d : d * ex2_approx(r);
      }
      warp_arrive(&bar->cumF[c & 1]);
      if (kShare) {
        const unsigned s = c & 1;
        wait(bar->cumF[s], c >> 1);
        wait(bar->fullX[s], c >> 1);
        if (a.cu != nullptr && it.t1 - it.t0 - (i64)c * kQ < kQ) wait(bar->xSync, 0);  // foreign rows are zeros
        const Cum& u = cum[s][WIDE ? 0 : q >> 1];
        const float one[4] = {1.f, 1.f, 1.f, 1.f};
        units.make(bar, tmem + lanes, s, 4 * c, u.u, ex2_approx(u.tot[1] + (u.tot[2] + u.tot[3])), one);
      }
    };
    if (PART) {
#pragma unroll 1
      for (unsigned c = 0; c < (unsigned)nblk; ++c) {
        if (c >= 2) wait(bar->xF[c & 1], (c >> 1) - 1);
        steps(c);
      }
    } else {
      if (nblk > 0) steps(0);
#pragma unroll 1
      for (unsigned c = 0; c < (unsigned)nblk; ++c) {
        const unsigned s = c & 1;
        wait(bar->cumF[s], c >> 1);
        const Cum* cu = cum[s];
        // M: this thread's row, 16 columns of each sub-block; the two warps
        // of a row share every sub-block, so the causal work is even.  16
        // fp32 columns become 8 + 8 columns of 16-bit pairs, one head each.
        constexpr int kH = WIDE ? 1 : 2;
        const uint32_t atG = tmem + lanes + kColG + 16 * hf;
        // While G runs: the row's own sum, its decay from the start of the
        // block (for inter), from the ends of the sub-blocks before its own.
        float l[kH], f[kH][3], e = 0.f;
#pragma unroll
        for (int k = 0; k < kH; ++k) {
          float sum = l[k] = cu[k].l[row];
#pragma unroll
          for (int b = 2; b >= 0; --b) {
            f[k][b] = ex2_approx(sum);
            if (b < q) sum += cu[k].tot[b];
          }
          if (k == hs) e = ex2_approx(sum);
        }
        wait(bar->gR, c);
        tc_after();
        {
          uint32_t v[16];
          tm_ld16(atG + 32 * q, v);
          tm_ld_wait();
          const int last = lane - 16 * hf;  // last unmasked column of the row's own sub-block
#pragma unroll
          for (int k = 0; k < kH; ++k) {
            const float4* lp = reinterpret_cast<const float4*>(cu[k].l + 32 * q + 16 * hf);
            const float4* dp = reinterpret_cast<const float4*>(cu[k].d + 32 * q + 16 * hf);
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 l4 = lp[j], d4 = dp[j];
              const float m0 = 4 * j + 0 <= last ? __uint_as_float(v[4 * j + 0]) * (ex2_approx(l[k] - l4.x) * d4.x) : 0.f;
              const float m1 = 4 * j + 1 <= last ? __uint_as_float(v[4 * j + 1]) * (ex2_approx(l[k] - l4.y) * d4.y) : 0.f;
              const float m2 = 4 * j + 2 <= last ? __uint_as_float(v[4 * j + 2]) * (ex2_approx(l[k] - l4.z) * d4.z) : 0.f;
              const float m3 = 4 * j + 3 <= last ? __uint_as_float(v[4 * j + 3]) * (ex2_approx(l[k] - l4.w) * d4.w) : 0.f;
              o[2 * j] = Pair<T>::pack(f2(m0, m1));
              o[2 * j + 1] = Pair<T>::pack(f2(m2, m3));
            }
            tm_st8(atG + 32 * q + 8 * k, o);
          }
        }
#pragma unroll
        for (int b = 0; b < 3; ++b) {
          if (b < q) {
            uint32_t v[16];
            tm_ld16(atG + 32 * b, v);
            tm_ld_wait();
#pragma unroll
            for (int k = 0; k < kH; ++k) {
              const float2 ff = f2(f[k][b], f[k][b]);
              const float4* up = reinterpret_cast<const float4*>(cu[k].u + 32 * b + 16 * hf);
              uint32_t o[8];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float4 w4 = up[j];
                o[2 * j] = Pair<T>::pack(mul2(mul2(f2(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])), f2(w4.x, w4.y)), ff));
                o[2 * j + 1] = Pair<T>::pack(mul2(mul2(f2(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])), f2(w4.z, w4.w)), ff));
              }
              tm_st8(atG + 32 * b + 8 * k, o);
            }
          }
        }
        {
          uint32_t v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = 0u;
#pragma unroll 1
          for (int b = q + 1; b < 4; ++b) tm_st16(atG + 32 * b, v);
        }
        // inter times exp(c_i), in place.
        const uint32_t atY = tmem + lanes + kColY + 64 * hf;
        wait(bar->iR, c);
        tc_after();
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
          uint32_t v[2][16];
          tm_ld16(atY + 32 * k, v[0]);
          tm_ld16(atY + 32 * k + 16, v[1]);
          tm_ld_wait();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float2 w = mul2(f2(__uint_as_float(v[h][j]), __uint_as_float(v[h][j + 1])), f2(e, e));
              v[h][j] = __float_as_uint(w.x);
              v[h][j + 1] = __float_as_uint(w.y);
            }
            tm_st16(atY + 32 * k + 16 * h, v[h]);
          }
        }
        tm_st_wait();
        tc_before();
        warp_arrive(&bar->pR);
        // The next block's steps, while intra runs.  Their stage is free: the
        // tokens' warps have read it before pR, the state's before xF, of the
        // block before.
        if (c + 1 < (unsigned)nblk) steps(c + 1);
        // y + D x, over x.
        wait(bar->yR, c);
        wait(bar->xF[s], c >> 1);
        tc_after();
        uint4* xr = reinterpret_cast<uint4*>(sm + kOffX + s * kTile + hf * kBox + row * 128);
        const int sw = row & 7;
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
          uint32_t v[2][16];
          tm_ld16(atY + 32 * k, v[0]);
          tm_ld16(atY + 32 * k + 16, v[1]);
          uint4 x4[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x4[j] = xr[(4 * k + j) ^ sw];
          tm_ld_wait();
          if (k == 1) {
            tc_before();
            warp_arrive(&bar->yF);  // inter of the next block may come
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t* wp = &x4[j].x;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const int o = 8 * (j & 1) + 2 * h;
              wp[h] = Pair<T>::pack(fma2(f2(Dh, Dh), Pair<T>::unpack(wp[h]),
                                         f2(__uint_as_float(v[j >> 1][o]), __uint_as_float(v[j >> 1][o + 1]))));
            }
            xr[(4 * k + j) ^ sw] = x4[j];
          }
        }
        fence_proxy_async_smem();
        warp_arrive(&bar->yS[s]);
        const i64 tb = it.t0 + (i64)c * kQ;
        if (a.cu != nullptr && it.t1 - tb < kQ) {
          // The last block of a packed sequence, in part: its rows only.
          wait(bar->yS[s], c >> 1);
          const int nv = (int)(it.t1 - tb);
          T* y = static_cast<T*>(a.y) + it.batch * a.ys_b + tb * a.ys_t + h0 * a.ys_h;
#pragma unroll 1
          for (int e = yt; e < 2 * kQ * 8; e += 256) {
            const int box = e >> 10, r = (e >> 3) & 127, un = e & 7;
            const int col = (WIDE ? 64 * box : 0) + 8 * un;
            if (r < nv && col < a.P && (WIDE || box < nh))
              *reinterpret_cast<uint4*>(y + r * a.ys_t + (WIDE ? 0 : box * a.ys_h) + col) =
                  *reinterpret_cast<const uint4*>(sm + kOffX + s * kTile + box * kBox + r * 128 + ((un ^ (r & 7)) << 4));
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
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
          if (a.init_f32) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (64 * hf + 4 * j < a.N) {
                const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(a.init) + o + 4 * j);
                S[4 * j] = v.x, S[4 * j + 1] = v.y, S[4 * j + 2] = v.z, S[4 * j + 3] = v.w;
              }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (64 * hf + 4 * j < a.N) {
                const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.init) + o + 4 * j);
                const float2 v0 = Pair<T>::unpack(v.x), v1 = Pair<T>::unpack(v.y);
                S[4 * j] = v0.x, S[4 * j + 1] = v0.y, S[4 * j + 2] = v1.x, S[4 * j + 3] = v1.y;
              }
          }
        }
#pragma unroll 1
        for (int r = 0; r < it.seg; ++r) {  // the earlier segments, in order
          const i64 slot = (part0 + (i64)r * part_step) * (WIDE ? 1 : 2) + hs;
          const float dc = ex2_approx(a.decay[slot]);
          const float* part = a.part + slot * a.P * a.N + e0;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (64 * hf + 4 * j < a.N) {
              const float4 v = *reinterpret_cast<const float4*>(part + 4 * j);
              S[4 * j] = fmaf(S[4 * j], dc, v.x), S[4 * j + 1] = fmaf(S[4 * j + 1], dc, v.y);
              S[4 * j + 2] = fmaf(S[4 * j + 2], dc, v.z), S[4 * j + 3] = fmaf(S[4 * j + 3], dc, v.w);
            }
        }
      }
    }
    float total = 0.f;   // base-2 log of the segment's decay
    const Units<T, TERMS> units(sm, q, hf, lane);
    float dec = 1.f, unscale = 1.f;
    // S = dec * S + dS of block c - 1 (c > 0), and with `copy` the 16-bit copy
    // of S for inter: row p, this thread's half of n.
    auto advance = [&](unsigned c, bool copy) {
      if (c > 0) {
        wait(bar->dR, c - 1);
        if (copy) wait(bar->iR, c - 1);  // inter has read the copy before
        tc_after();
      }
      uint4* sr = reinterpret_cast<uint4*>(sm + kOffS + hf * kBox + row * 128);
      const float2 dd = f2(dec, dec), uu = f2(unscale, unscale);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (c > 0 && hf < p.nb) {
          uint32_t v[2][16];
          tm_ld16(tmem + lanes + kColD + 64 * hf + 32 * k, v[0]);
          tm_ld16(tmem + lanes + kColD + 64 * hf + 32 * k + 16, v[1]);
          tm_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 n = fma2(f2(S[32 * k + j], S[32 * k + j + 1]), dd,
                                  mul2(f2(__uint_as_float(v[j >> 4][j & 15]), __uint_as_float(v[j >> 4][(j & 15) + 1])), uu));
            S[32 * k + j] = n.x;
            S[32 * k + j + 1] = n.y;
          }
        }
        if (copy) {
#pragma unroll
          for (int j = 4 * k; j < 4 * k + 4; ++j) {
            uint4 w;
            w.x = Pair<T>::pack(f2(S[8 * j], S[8 * j + 1]));
            w.y = Pair<T>::pack(f2(S[8 * j + 2], S[8 * j + 3]));
            w.z = Pair<T>::pack(f2(S[8 * j + 4], S[8 * j + 5]));
            w.w = Pair<T>::pack(f2(S[8 * j + 6], S[8 * j + 7]));
            sr[j ^ (row & 7)] = w;
          }
        }
      }
      if (c > 0) {
        tc_before();
        warp_arrive(&bar->dF);
      }
      if (copy) {
        fence_proxy_async_smem();
        warp_arrive(&bar->sR);
      }
    };
#pragma unroll 1
    for (unsigned c = 0; c < (unsigned)nblk; ++c) {
      const unsigned s = c & 1;
      wait(bar->fullX[s], c >> 1);
      unsigned char* xt = sm + kOffX + s * kTile;
      const i64 tb = it.t0 + (i64)c * kQ;
      if (a.cu != nullptr && it.t1 - tb < kQ) {
        // The rows behind the sequence's end belong to others, whatever they
        // hold: zeros keep it out of the sums.
        wait(bar->fullB[s], c >> 1);
        const int nv = (int)(it.t1 - tb);
#pragma unroll 1
        for (int e = nv * 8 + st; e < kQ * 8; e += 256) {
          const uint4 z = make_uint4(0u, 0u, 0u, 0u);
          reinterpret_cast<uint4*>(xt)[e] = z;
          reinterpret_cast<uint4*>(xt + kBox)[e] = z;
          for (int k = 0; k < p.nb; ++k) reinterpret_cast<uint4*>(sm + kOffB + s * kTile + k * kBox)[e] = z;
        }
        fence_proxy_async_smem();
        warp_arrive(&bar->xSync);
        wait(bar->xSync, 0);  // a sequence has one such block, its last
      }
      wait(bar->cumF[s], c >> 1);
      const Cum& u = cum[s][hs];
      // Decay from the end of each sub-block to the block's end, of the whole block.
      const float after2 = u.tot[3], after1 = u.tot[2] + after2, after0 = u.tot[1] + after1;
      const float g0 = ex2_approx(after0), g1 = ex2_approx(after1), g2 = ex2_approx(after2);
      float scale[4] = {1.f, 1.f, 1.f, 1.f}, next_unscale = 1.f;
      const float next_dec = ex2_approx(u.tot[0] + after0);
      if (kRowScale<T>) {
        // The largest |w x| of each row, of both its warps.
        float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (unsigned un = 0; un < 4; ++un) {
          uint32_t x[8];
          units.load(s, un, x);
          const float g = un == 0 ? g0 : un == 1 ? g1 : un == 2 ? g2 : 1.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 w = *reinterpret_cast<const float2*>(u.u + units.token + 32 * un + 4 * (i & 2));
            const float2 v = mul2(mul2(w, f2(g, g)), Pair<T>::unpack(x[i]));
            m[2 * (i >> 2) + (i & 1)] = fmaxf(m[2 * (i >> 2) + (i & 1)], fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        }
        float* rm = reinterpret_cast<float*>(sm + kOffMax);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m[i] = fmaxf(m[i], __shfl_xor_sync(kFull, m[i], 1));
          m[i] = fmaxf(m[i], __shfl_xor_sync(kFull, m[i], 2));
          if ((lane & 3) == 0) rm[hf * kQ + q * 32 + 8 * i + (lane >> 2)] = m[i];
        }
        warp_arrive(&bar->mSync);
        wait(bar->mSync, c);
        auto exponent = [&](int r) { return max((__float_as_uint(fmaxf(rm[r], rm[kQ + r])) >> 23) & 255u, 15u); };
#pragma unroll
        for (int i = 0; i < 4; ++i)
          scale[i] = __uint_as_float((268u - exponent(q * 32 + 8 * i + (lane >> 2))) << 23);  // the largest into [2^14, 2^15)
        next_unscale = __uint_as_float((exponent(row) - 14u) << 23);
      }
#pragma unroll 1
      for (unsigned un = kShare ? 1 : 0; un < 4; ++un) {
        // The state of the block before, as soon as its last unit is through.
        if (un == 1) advance(c, !PART);
        const float g = un == 0 ? g0 : un == 1 ? g1 : un == 2 ? g2 : 1.f;
        units.make(bar, tmem + lanes, s, 4 * c + un, u.u, g, scale);
      }
      if (PART) total += u.tot[0] + after0;
      warp_arrive(&bar->xF[s]);  // x and the steps have been read
      dec = next_dec;
      unscale = next_unscale;
    }
    if (nblk > 0) advance(nblk, false);
    float* out = nullptr;
    if (live) {
      const i64 h = h0 + hs;
      if (PART) {
        const i64 slot = (part0 + (i64)it.seg * part_step) * (WIDE ? 1 : 2) + hs;
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
  __syncwarp();
  tc_before();
  __syncthreads();
  if (threadIdx.x == 0 && *(volatile int*)&bar->abort) atomicAdd(&g_cc1d_wait_timeouts, 1u);
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
  const i64 grid = t.a.cu ? t.a.items * t.npairs : (PART ? 0 : t.a.whole) + ((i64)t.a.nseq * t.npairs - t.a.whole) * t.a.segs;
  return launch_pdl(scan_tc_kernel<T, TERMS, PART, WIDE>, dim3((unsigned)grid), dim3(kThreads), kSmem, s, t);
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

i64 scan_tc_parts(const ScanArgs& a) {
  const i64 pairs = scan_tc_pairs(a);
  return (a.cu ? a.items * pairs : (a.nseq * pairs - a.whole) * a.segs) * (a.P > 64 ? 1 : 2);
}

bool scan_tc_eligible(int dtype, const ScanArgs& a, i64 batch) {
  if (dtype == 2 || a.P < 8 || a.P > 128 || a.P % 8 || a.N < 8 || a.N > 128 || a.N % 8) return false;
  return tile_ok(a.x, a.xs_p, a.H, a.xs_h, a.L, a.xs_t, batch, a.xs_b) &&
         tile_ok(a.B, a.bs_n, a.G, a.bs_g, a.L, a.bs_t, batch, a.bs_b) &&
         tile_ok(a.C, a.cs_n, a.G, a.cs_g, a.L, a.cs_t, batch, a.cs_b) &&
         tile_ok(a.y, 1, a.H, a.ys_h, a.L, a.ys_t, batch, a.ys_b) &&
         (a.init == nullptr || (reinterpret_cast<uintptr_t>(a.init) % 16 == 0 && a.is_s % 4 == 0 && a.is_h % 4 == 0)) &&
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
      !make_map(&t.my, bf, a.y, a.P, a.H, a.L, batch, a.ys_h, a.ys_t, a.ys_b) ||
      !make_map(&t.mc, bf, a.C, a.N, a.G, a.L, batch, a.cs_g, a.cs_t, a.cs_b))
    return cudaErrorInvalidValue;
  if (bf) return wide ? launch_all<__nv_bfloat16, true>(t, stream) : launch_all<__nv_bfloat16, false>(t, stream);
  return wide ? launch_all<__half, true>(t, stream) : launch_all<__half, false>(t, stream);
}

cudaError_t read_scan_wait_timeouts(unsigned* count) { return tu_read_wait_timeouts(count); }

}  // namespace cc1d
