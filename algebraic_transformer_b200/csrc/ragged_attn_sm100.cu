// Causal asinh-power attention over sequences of different lengths, grouped heads, keys packed or in pages: tcgen05.
//
//   w_ij = rho(x_ij)^n, x = q.k / (sqrt(D) c), j <= i + Lk - Lq;  l_i = rho(b/c)^n + sum_j w_ij;  o_i = sum_j w_ij v_j / l_i
//
// The arithmetic per tile is that of attn_sm100.cu: S = Q K^T as 128 x 128 products, (y + sqrt(kappa + y^2))^n on packed fp32
// straight from tensor memory (Q carries the power of two of the score scale), P back over S, O += P V with P from tensor
// memory.  What is different:
//   - work comes from a list made on the device (ragged.cuh, ragged_plan.cu), taken from a counter, and handed round the CTA
//     through a small ring;
//   - a query tile's rows are G heads of 128 / G tokens;
//   - K and V tiles come from packed rows (a tile reads on into the next sequence) or page by page through the block table.
//     Keys past the sequence's end are masked by the causal limit, but 0 times the NaN or infinity that a
//     foreign V row may hold is NaN: one warp zeroes those rows of a sequence's last V tile in shared memory;
//   - any scores: a warp takes a tile unshifted where all its |x| <= x_fast (which keeps the weights within 2^+-64 and the
//     cancellation of y + sqrt(kappa + y^2) below 3.3e-4 of a weight).  For packed keys the largest row norms of the call's keys (ragged_plan.cu) and
//     of the item's queries settle that as a rule; else the scores are looked at ahead of their weights: a sum of squares, then the largest.  A
//     score out of range, or a NaN, sends the warp to the max-shifted form with the cancellation-free rho for the rest of the item;
//   - values of any size: unshifted weights go up to 2^64 and may take the sum of finite values out of range.  A row that comes out
//     infinite or NaN with finite weights has its item noted; when the list is done the CTA takes its noted items once more,
//     max-shifted from the first tile on (weights of 1 at most), and writes the rows again that had come out so.
//
// Roles: warp 0 takes the work and runs the TMA loads, warp 1 issues the MMAs, warp 2 scales Q in shared memory and takes its row norms, warp 3 clears the
// foreign V rows, warps 4..7 and 8..11 weigh query tile 0 and 1, a thread a row.  An item of one tile runs as tile 1.
// HILO (training): the weights go to the second product as two bf16 halves and the output is stored as two, for delta = dO . o, which the
// backward takes from dP where p has nearly all of a row: with 8 bits of either, dq and dk are off by 0.0029 (normalised rows), 0.0048 (scores four
// times as large) and 0.0052 (nine times) of their norm against 64 bits, with 16 bits by 0.0024 throughout, which is the rounding of dS.
//
// Measured, with the plan ahead: 24 prompts of 19 to 2001 tokens, 16 heads on 4 of 64: 95 us; two of 5623 and 8192, 16 on 2 of 128: 431 us,
// 937 TFLOP/s; chunks of 620 and 2048 tokens on caches of 24784 and 30001 keys, 16 on 4 of 128: 681 us, 897 TFLOP/s.  No pipe is full (MUFU 37 %,
// FMA 34 %, tensor 20 % in the first): the chain scores -> weights -> P V -> next scores through tensor memory and barriers is what it
// waits for; with the weights' arithmetic left out it still took 72 of 92 us, 356 of 427.
//
// Every mbarrier wait is bounded; a wait that runs out reports ALG_DEV_TIMEOUT, and the rows of the items that its CTA had not finished, and of those
// that no CTA had taken by then, are NaN.
#include "common.cuh"
#include "launchers.h"
#include "ragged.cuh"
#include "sm100_ptx.cuh"

#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

namespace alg {
namespace {

using namespace sm100;

constexpr int BQ = 128, BKEY = 128;
constexpr int FIRST_WEIGHT_WARP = 4, NTHREADS = 384;
constexpr int PANEL_BYTES = 128 * 128;          // 128 rows x 64 bf16, one swizzle-128B panel
constexpr uint32_t TMEM_COLS = 512;
constexpr int MAX_NKV = 10, RING = 3;
constexpr int ITEM_READERS = 11;                // warps 1..11
static_assert(NTHREADS / 32 % 4 == 0, "the warps are dealt over the panels of two query tiles");

template <int D> struct Cfg {
  static constexpr int PANELS = D / 64;
  static constexpr int TILE_BYTES = PANELS * PANEL_BYTES;
  static constexpr int NKV = (D == 128) ? 5 : 10;           // K/V ring depth (tiles)
  static constexpr int KV_OFF = 2 * TILE_BYTES;             // behind the two Q tiles
  static constexpr int CTL_OFF = KV_OFF + NKV * TILE_BYTES;
  static constexpr uint32_t IDESC_S = make_idesc_bf16(BQ, BKEY, 0, 0);
  static constexpr uint32_t IDESC_PV = make_idesc_bf16(BQ, D, 0, 1);   // V is [key][d]: MN-major B
};

// What a work item is to the roles.
struct Work {
  int row0, Lq, Lk, seq;
  int head;                       // key head
  int tok0, tok1;                 // first token (in the sequence) of query tile 0 / 1
  int k0, n0, n1;                 // first key tile; key tiles of query tile 0 (0: it has none in this item) and 1 (< 0: no more work)
  int has0;                       // query tile 0 has tokens
  int slot;                       // < 0: whole
  int index;                      // its place in the list, times Hkv, plus the head
};

struct Barriers {
  uint64_t q_full[2], q_ready[2], q_free[2], kv_full[MAX_NKV], kv_empty[MAX_NKV];
  uint64_t s_full[2], p_half[2], p_full[2], o_full[2], o_free[2];
  uint64_t q_norm_full[2], v_here, v_clean, never, work_full[RING], work_empty[RING];
};
struct __align__(16) Control {
  Barriers bars[2];               // of the first pass and of the second (one set, invalidated and set up again, kept the phase of its last barrier)
  Work work[RING];
  float q_norm[2][2];             // largest squared row norm of a query tile, of this item and the next one
  int overflowed[RING];           // a row of the item came out infinite or NaN
  int taken, noted;               // items that this CTA has taken; those of them that it has looked at for the word above
  int again;                      // the last item to be weighed again; -1: none
  uint32_t tmem_base;
  int abort_flag;
};

template <int D> constexpr size_t smem_bytes() { return size_t(Cfg<D>::CTL_OFF) + sizeof(Control) + 1024; }
static_assert(smem_bytes<128>() <= 232448 && smem_bytes<64>() <= 232448, "shared memory budget of one CTA");

struct ScoreScale {
  float pow2;      // 2^e: applied to Q in shared memory
  float m;         // x = m y
  float kappa;     // 1 / m^2
  float inv_m;     // every weight is (rho(x) / m)^n
  float y_fast;    // x_fast / m
};

// 32 weights of this thread's row into bf16 pairs, hi and (HILO) what the rounding left over
template <bool HILO>
__device__ __forceinline__ void pack4(float2 t0, float2 t1, int i, uint32_t* packed) {
  const uint32_t h0 = pack_bf16(t0.x, t0.y), h1 = pack_bf16(t1.x, t1.y);
  packed[i >> 1] = h0;
  packed[(i >> 1) + 1] = h1;
  if (HILO) {
    packed[16 + (i >> 1)] = pack_bf16(t0.x - __uint_as_float(h0 << 16), t0.y - __uint_as_float(h0 & 0xffff0000u));
    packed[16 + (i >> 1) + 1] = pack_bf16(t1.x - __uint_as_float(h1 << 16), t1.y - __uint_as_float(h1 & 0xffff0000u));
  }
}
template <bool HILO> __device__ __forceinline__ void store_packed(uint32_t taddr, const uint32_t* packed) {
  if (HILO) tmem_st_32x32(taddr, packed);
  else tmem_st_32x16(taddr, packed);
}

// Unshifted: 32 scores y -> (y + sqrt(kappa + y^2))^n.  `lim`: the last visible column of this row, counted from column 0 of the 32.  Formed
// in passes over PAIRS pairs, so that every pass has independent operations: with two warps on a scheduler nothing else hides their latency.
template <int LOG2N, bool MASK, bool HILO>
__device__ __forceinline__ void weigh(const uint32_t* s, float kappa, int log2n, int lim, float2& la, float2& lb, uint32_t* packed) {
  constexpr int PAIRS = 8;
  const float2 kp = make_float2(kappa, kappa);
#pragma unroll
  for (int i0 = 0; i0 < 32; i0 += 2 * PAIRS) {
    float2 t[PAIRS];
    {
      float2 rad[PAIRS];
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 y = make_float2(__uint_as_float(s[i0 + 2 * i]), __uint_as_float(s[i0 + 2 * i + 1]));
        rad[i] = __ffma2_rn(y, y, kp);
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) t[i] = make_float2(rsqrt_approx(rad[i].x), rsqrt_approx(rad[i].y));
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) t[i] = __ffma2_rn(rad[i], t[i], make_float2(__uint_as_float(s[i0 + 2 * i]), __uint_as_float(s[i0 + 2 * i + 1])));
    }
    if (LOG2N > 0) {
#pragma unroll
      for (int k = 0; k < LOG2N; ++k)
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) t[i] = __fmul2_rn(t[i], t[i]);
    } else {
      for (int k = 0; k < log2n; ++k)
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) t[i] = __fmul2_rn(t[i], t[i]);
    }
#pragma unroll
    for (int i = 0; i < PAIRS; i += 2) {
      if (MASK) {
        t[i].x = (i0 + 2 * i <= lim) ? t[i].x : 0.f;             t[i].y = (i0 + 2 * i + 1 <= lim) ? t[i].y : 0.f;
        t[i + 1].x = (i0 + 2 * i + 2 <= lim) ? t[i + 1].x : 0.f; t[i + 1].y = (i0 + 2 * i + 3 <= lim) ? t[i + 1].y : 0.f;
      }
      la = __fadd2_rn(la, t[i]);
      lb = __fadd2_rn(lb, t[i + 1]);
      pack4<HILO>(t[i], t[i + 1], i0 + 2 * i, packed);
    }
  }
}

// Shifted: (rho(x) sigma)^n with the cancellation-free rho, x = m y; sigma = rho(-reference) / m.
template <bool HILO>
__device__ __forceinline__ void weigh_shifted(const uint32_t* s, float m, float sigma, int log2n, int lim, float2& la, float2& lb,
                                              uint32_t* packed) {
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    float t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = __uint_as_float(s[i + e]) * m, rad = fmaf(x, x, 1.0f);
      float T = fmaf(rad, rsqrt_approx(rad), fabsf(x));
      T = rad < 3.0e38f ? T : 2.0f * fabsf(x);           // x^2 past the range: sqrt(1 + x^2) = |x|
      t[e] = pow2n_rt((x >= 0.f ? T : __fdividef(1.0f, T)) * sigma, log2n);
      t[e] = (i + e <= lim) ? t[e] : 0.f;
    }
    const float2 t0 = make_float2(t[0], t[1]), t1 = make_float2(t[2], t[3]);
    la = __fadd2_rn(la, t0);
    lb = __fadd2_rn(lb, t1);
    pack4<HILO>(t0, t1, i, packed);
  }
}
// What this warp has done with tensor memory is done: one arrival a warp.  (An arrival a thread is 32 operations on one word of
// shared memory, two or three times a tile.)
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ void signal_weights(uint64_t* bar) {
  tmem_st_wait();
  warp_arrive(bar);
}

// Sum of y^2 over the row's 128 scores, whatever the mask: where it is within the square of the range, so is every score.
__device__ __forceinline__ float tile_square_sum(uint32_t s_taddr) {
  uint32_t a[32], b[32];
  float2 m0 = make_float2(0.f, 0.f), m1 = make_float2(0.f, 0.f);
  auto add = [&](const uint32_t* s) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float2 y0 = make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), y1 = make_float2(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
      m0 = __ffma2_rn(y0, y0, m0);
      m1 = __ffma2_rn(y1, y1, m1);
    }
  };
  tmem_ld_32x32(s_taddr, a);
  tmem_ld_32x32(s_taddr + 32, b);
  tmem_ld_wait_for(a);
  tmem_ld_wait_for(b);                                  // complete already: orders the reads of b
  add(a);
  tmem_ld_32x32(s_taddr + 64, a);
  add(b);
  tmem_ld_32x32(s_taddr + 96, b);
  tmem_ld_wait_for(a);
  add(a);
  tmem_ld_wait_for(b);
  add(b);
  return (m0.x + m0.y) + (m1.x + m1.y);
}
// Largest |y| of the row's visible scores, NaN if one is NaN.  Only what the row sees counts: which form its weights take, and
// with it their rounding, must not depend on a neighbouring sequence.
__device__ __forceinline__ float tile_abs_max(uint32_t s_taddr, int lim) {
  float most = 0.f;
#pragma unroll 1
  for (int c = 0; c < 128; c += 32) {
    uint32_t a[32];
    tmem_ld_32x32(s_taddr + c, a);
    tmem_ld_wait_for(a);
#pragma unroll
    for (int i = 0; i < 32; i += 2)
      most = max3_abs_nan(most, c + i <= lim ? __uint_as_float(a[i]) : 0.f, c + i + 1 <= lim ? __uint_as_float(a[i + 1]) : 0.f);
  }
  return most;
}

// The unshifted weights of a tile, written over the scores, the next 32 scores in flight while a block is weighed.  A loop of two times
// two blocks: unrolled, the tile is more code than two warps that are not at the same place in it find in the SM's instruction caches
// (97 against 94 us for 24 prompts, 16 heads on 4 of 64).  Weights in columns of their own, so that the next scores could be issued
// as soon as these are read, were no faster (94 against 92), nor were all 128 scores in registers.
template <int LOG2N, bool HILO>
__device__ __forceinline__ void weigh_tile(uint32_t s_taddr, uint64_t* p_half, uint64_t* p_full, float kappa, int log2n, int lim, bool masked,
                                           float2& la, float2& lb) {
  uint32_t a[32], b[32], packed[HILO ? 32 : 16];
  const int warp_lim = masked ? __reduce_max_sync(0xffffffffu, lim) : 128;
  auto block = [&](const uint32_t* s, int c) {
    if (!masked) {
      weigh<LOG2N, false, HILO>(s, kappa, log2n, 0, la, lb, packed);
    } else if (c <= warp_lim) {
      weigh<LOG2N, true, HILO>(s, kappa, log2n, lim - c, la, lb, packed);
    } else {                                            // the block lies beyond what any row of the warp sees
#pragma unroll
      for (int i = 0; i < (HILO ? 32 : 16); ++i) packed[i] = 0u;
    }
  };
  tmem_ld_32x32(s_taddr, a);
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    tmem_ld_wait_for(a);
    tmem_ld_32x32(s_taddr + 32, b);
    block(a, 64 * half);
    store_packed<HILO>(s_taddr, packed);
    tmem_ld_wait_for(b);
    if (half == 0) tmem_ld_32x32(s_taddr + 64, a);
    block(b, 64 * half + 32);
    store_packed<HILO>(s_taddr + 32, packed);
    signal_weights(half == 0 ? p_half : p_full);
    s_taddr += 64;
  }
}

// The max-shifted form reads the scores again from tensor memory, block by block: it runs where the short form may not, and
// its code stays small.
// Largest visible x of the row (NaN ignored: its weight will be NaN whatever the reference); -inf if there is none.
__device__ __forceinline__ float tile_row_max(uint32_t s_taddr, float m, int lim) {
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 128; c += 32) {
    uint32_t a[32];
    tmem_ld_32x32(s_taddr + c, a);
    tmem_ld_wait_for(a);
#pragma unroll
    for (int i = 0; i < 32; ++i) top = (c + i <= lim) ? fmaxf(top, __uint_as_float(a[i]) * m) : top;
  }
  return top;
}
template <bool HILO>
__device__ __forceinline__ void weigh_tile_shifted(uint32_t s_taddr, uint64_t* p_half, uint64_t* p_full, float m, float sigma,
                                                   int log2n, int lim, float2& la, float2& lb) {
#pragma unroll 1
  for (int b = 0; b < 4; ++b) {
    uint32_t a[32], packed[HILO ? 32 : 16];
    tmem_ld_32x32(s_taddr + 32 * b, a);
    tmem_ld_wait_for(a);
    weigh_shifted<HILO>(a, m, sigma, log2n, lim - 32 * b, la, lb, packed);
    store_packed<HILO>(s_taddr + 32 * b, packed);
    if (b == 1) signal_weights(p_half);
  }
  signal_weights(p_full);
}

// Largest squared norm of a query tile's 128 rows, a little above the true one: squares are added up in bf16, D / 8 of them to a sum, each
// sum off by a half step at most.  NaN or infinity where a row holds one.
template <int D> __device__ __forceinline__ float largest_row_norm(const unsigned char* tile, int lane) {
  float most = 0.f;
#pragma unroll 1
  for (int r = lane; r < 128; r += 32) {
    __nv_bfloat162 sum[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = __float2bfloat162_rn(0.f);
#pragma unroll
    for (int pn = 0; pn < D / 64; ++pn)
#pragma unroll
      for (int c = 0; c < 8; ++c) {                    // chunks in an order of the row's own: no two of eight lanes in one bank group
        const uint4 v = *reinterpret_cast<const uint4*>(tile + pn * PANEL_BYTES + r * 128 + ((c ^ (r & 7)) << 4));
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = __hfma2(h[e], h[e], sum[e]);
      }
    float n = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) { const float2 f = __bfloat1622float2(sum[e]); n += f.x + f.y; }
    most = max3_abs_nan(most, n, 0.f);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max3_abs_nan(most, __shfl_xor_sync(0xffffffffu, most, o), 0.f);
  return most * 1.07f;                                 // (1 - 2^-9)^-16 and the sum of the eight
}

constexpr float FLT_LARGEST = 0x1.fffffep127f, BF16_INFINITE = 0x1.ffp127f;     // the latter and what is larger round to infinity
// Is one of the row's D numbers infinite or NaN?
template <int D> __device__ __forceinline__ bool any_not_finite(const float* row) {
  float most = 0.f;
#pragma unroll 1
  for (int i = 0; i < D; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(row + i);
    most = max3_abs_nan(max3_abs_nan(most, v.x, v.y), v.z, v.w);
  }
  return !(most <= FLT_LARGEST);
}
template <int D> __device__ __forceinline__ bool any_not_finite(const __nv_bfloat16* row) {
  bool any = false;
#pragma unroll 1
  for (int i = 0; i < D; i += 2) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + i);
    any |= (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
  }
  return any;
}

template <int NKV> struct RingCursor {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() { if (++slot == NKV) { slot = 0; phase ^= 1u; } }
};

// NaN to this thread's row of an item that has no result and will get none; a weight warp's threads.
template <int D, bool HILO> __device__ __noinline__ void spoil_row(const RaggedParams& p, const Work& w, int warp, int lane) {
  const int t = (warp - FIRST_WEIGHT_WARP) >> 2, r = (warp & 3) * 32 + lane, tok_r = r / p.G, head = w.head * p.G + r - tok_r * p.G;
  const int tok = (t == 0 ? w.tok0 : w.tok1) + tok_r;
  if (tok_r >= p.tile_tokens || tok >= w.Lq || (t == 0 && w.has0 == 0)) return;
  const float nan = __int_as_float(0x7fc00000);
  if (w.slot >= 0) {
    float* dst = p.plan.slots + ((int64_t(w.slot) * p.Hkv + w.head) * 256 + t * BQ + r) * (D + 4);
    *reinterpret_cast<float4*>(dst + D) = make_float4(nan, 0.f, 0.f, 0.f);
    return;
  }
  const int64_t row = int64_t(w.row0) + tok;
#pragma unroll 1
  for (int c = 0; c < D; c += 8) {
    const uint4 v = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.o) + row * p.os.t + head * p.os.h + c) = v;
    if (HILO) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.o_lo) + (row * p.H + head) * D + c) = v;
  }
  if (p.stat != nullptr) p.stat[int64_t(head) * p.seqs.tokens + row] = nan;
}

template <int D, int LOG2N, bool HILO, bool PAGED>
__global__ void __launch_bounds__(NTHREADS, 1)
ragged_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ RaggedParams p, const ScoreScale sc) {
  using C = Cfg<D>;
  constexpr bool NORMS = !PAGED;
  constexpr uint32_t O_COL = 256;                       // tensor memory: S_t at 128 t with P_t inside it, O_t at O_COL + D t
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Control* ctl = reinterpret_cast<Control*>(smem + C::CTL_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (lane == 0 && (warp == 0 || warp == 3)) {
    Barriers* bar = &ctl->bars[warp == 0 ? 0 : 1];
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bar->q_full[w], 1); mbar_init(&bar->q_ready[w], 1); mbar_init(&bar->q_free[w], NORMS ? 5 : 1);
      mbar_init(&bar->s_full[w], 1); mbar_init(&bar->p_half[w], 4); mbar_init(&bar->p_full[w], 4);
      mbar_init(&bar->o_full[w], 1); mbar_init(&bar->o_free[w], 4);
      mbar_init(&bar->q_norm_full[w], 1);
    }
    for (int i = 0; i < C::NKV; ++i) { mbar_init(&bar->kv_full[i], 1); mbar_init(&bar->kv_empty[i], 1); }
    for (int i = 0; i < RING; ++i) { mbar_init(&bar->work_full[i], 1); mbar_init(&bar->work_empty[i], ITEM_READERS); }
    mbar_init(&bar->v_here, 1); mbar_init(&bar->v_clean, 1); mbar_init(&bar->never, 1);
    fence_barrier_init();
  }
  if (threadIdx.x == 0) {
    ctl->abort_flag = 0;
    ctl->taken = ctl->noted = 0;
    ctl->again = -1;
    tma_prefetch_desc(&tm_q); tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  // Rows of a query tile that no load writes, where G does not divide 128: zeros.  What a kernel before left there would have its say in
  // the tile's row norm, and a NaN or a large number cost every item of the CTA the look at its scores (61.5 against 58.4 us for eight
  // prompts of 300 to 2001, 12 heads on 4 of 64).
  const int TT = p.tile_tokens;
  if (const int loaded = p.G * TT; loaded < 128) {
    const int panel = warp % (2 * C::PANELS);
    for (int r = loaded + warp / (2 * C::PANELS); r < 128; r += NTHREADS / 32 / (2 * C::PANELS))
      if (lane < 8) reinterpret_cast<uint4*>(smem + panel * PANEL_BYTES + r * 128)[lane] = make_uint4(0u, 0u, 0u, 0u);
    fence_async_shared();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_wait();                                       // the plan, and q, k, v of the kernels ahead
  const uint32_t tmem_base = ctl->tmem_base;
  const BoundedWait bw{&ctl->abort_flag, 1000000000ull};

  // item `next` of the list of `total`; false behind its end
  auto item_at = [&](int next, int total, Work& w) -> bool {
    w.n1 = -1;
    if (next >= total) return false;
    const RaggedItem it = p.plan.items[next / p.Hkv];
    w.index = next;
    w.head = next % p.Hkv;
    w.row0 = it.row0; w.Lq = it.Lq; w.Lk = it.Lk; w.seq = it.seq; w.k0 = it.k0; w.slot = it.slot; w.n1 = it.nk;
    const bool two = it.Lq - it.t0 > TT;
    w.has0 = two ? 1 : 0;
    w.tok0 = it.t0;
    w.tok1 = two ? it.t0 + TT : it.t0;
    w.n0 = two ? min(max(ragged_tiles(it.Lq, it.Lk, it.t0 + TT) - it.k0, 0), it.nk) : 0;
    return true;
  };
  // the oldest item that has not been looked at; all roles are done with it
  auto note = [&] {
    const int k = ctl->noted++ % RING;
    if (ctl->overflowed[k] == 0) return;
    p.plan.again[ctl->work[k].index] = ctl->again;
    ctl->again = ctl->work[k].index;
  };

  int undone = 0;                                       // weight warps: items of the first pass that they have finished
  auto run = [&](auto again) {                          // the list; again: the noted items, in a copy of its own that costs the first nothing
    constexpr bool SECOND = decltype(again)::value;
    Barriers* const bar = &ctl->bars[SECOND ? 1 : 0];
    // the k-th work item of this CTA; false at the end of the work or of the waiting
    auto work_at = [&](int k, Work& w) -> bool {
      if (!__all_sync(0xffffffffu, bw.wait(&bar->work_full[k % RING], uint32_t(k / RING) & 1u))) return false;
      w = ctl->work[k % RING];
      return w.n1 >= 0;
    };
    auto work_done = [&](int k) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->work_empty[k % RING]);
    };
    if (warp == 0) {
      if (lane == 0) {
        const int total = p.plan.header->items * p.Hkv;
        // the next item: the CTA's own number first, then from the counter; shown to the other roles.  It is asked for when the loads of
        // the item before have been issued, which is as late as can be without a pause, so that longest-first holds to the end
        auto fetch = [&](int k, Work& w) -> bool {
          if (k >= RING && !bw.wait(&bar->work_empty[k % RING], uint32_t(k / RING - 1) & 1u)) return false;
          int next;
          if (!SECOND) {
            if (k >= RING) note();
            next = k == 0 ? int(blockIdx.x) : int(gridDim.x) + atomicAdd(&p.plan.header->counter, 1);
          } else {
            next = ctl->again < 0 ? INT_MAX : ctl->again;
            if (ctl->again >= 0) ctl->again = p.plan.again[next];
          }
          if (item_at(next, total, w)) {
            ctl->overflowed[k % RING] = 0;
            ++ctl->taken;
          }
          ctl->work[k % RING] = w;
          mbar_arrive(&bar->work_full[k % RING]);
          return w.n1 >= 0;
        };
        RingCursor<C::NKV> cur;
        int items0 = 0;                                   // items in which query tile 0 took part
        int left = p.limits.max_loads;                    // K and V tiles that it may load
        Work w;
        bool ok = true;
        for (int k = 0; ok && fetch(k, w); ++k) {
          auto load_kv = [&](int idx) {                   // K_0, V_0, K_1, V_1, ... of this item
            const int buf = cur.slot;
            if (!bw.wait(&bar->kv_empty[buf], cur.phase ^ 1u)) return false;
            const CUtensorMap* tm = (idx & 1) ? &tm_v : &tm_k;
            unsigned char* dst = smem + C::KV_OFF + buf * C::TILE_BYTES;
            const int key0 = (w.k0 + (idx >> 1)) * BKEY;
            if (PAGED) {
              const int rows = min(p.page, BKEY), live = min(BKEY, w.Lk - key0);      // keys of the tile that the sequence has
              const int loads = live > 0 ? (live + rows - 1) / rows : 0;
              mbar_arrive_expect_tx(&bar->kv_full[buf], uint32_t(loads * rows) * (D * 2));
              const int* pages = p.table + w.seq * p.table_stride;
              for (int i = 0; i < loads; ++i) {
                const int key = key0 + i * rows;
                const int number = __ldg(pages + (key >> p.log2_page));    // outside the pool: the copy fills zeros
                for (int pn = 0; pn < C::PANELS; ++pn)
                  tma_load_5d(dst + pn * PANEL_BYTES + i * rows * 128, tm, &bar->kv_full[buf], 0, key & (p.page - 1), pn, w.head, number);
              }
            } else {
              mbar_arrive_expect_tx(&bar->kv_full[buf], C::TILE_BYTES);
              tma_load_4d(dst, tm, &bar->kv_full[buf], 0, w.row0 + key0, 0, w.head);
            }
            cur.next();
            return true;
          };
          auto load_q = [&](int t) {                      // after the previous item's last S_t has read the tile
            if (t == 0 && w.n0 == 0) return true;
            const int before = t == 0 ? items0 : k;
            if (before > 0 && !bw.wait(&bar->q_free[t], uint32_t(before - 1) & 1u)) return false;
            mbar_arrive_expect_tx(&bar->q_full[t], uint32_t(p.G * TT) * (D * 2));
            for (int pn = 0; pn < C::PANELS; ++pn)
              tma_load_4d(smem + t * C::TILE_BYTES + pn * PANEL_BYTES, &tm_q, &bar->q_full[t], 0, w.head * p.G,
                          w.row0 + (t == 0 ? w.tok0 : w.tok1), pn);
            return true;
          };
          const int loads = min(2 * w.n1, left);
          left -= loads;
          if (loads < 2) ok = false;
          else if (k == 0) ok = load_q(0) && load_kv(0) && load_q(1) && load_kv(1);
          else ok = load_kv(0) && load_q(0) && load_kv(1) && load_q(1);
          for (int idx = 2; idx < loads && ok; ++idx) ok = load_kv(idx);
          if (loads < 2 * w.n1) ok = wait_in_vain(&ctl->abort_flag, &bar->never, p.limits.budget_ns);
          if (w.n0 > 0) ++items0;
        }
      }
    } else if (warp == 1) {
      const uint32_t q_addr = smem_u32(smem), kv_addr = smem_u32(smem + C::KV_OFF);
      using Cur = RingCursor<C::NKV>;
      Cur cur;
      int t0 = 0, t1 = 0, items0 = 0, cleans = 0;         // score tiles of query tile 0 / 1 in earlier items; items of tile 0
      auto wait_all = [&](uint64_t* word, uint32_t parity) { return __all_sync(0xffffffffu, bw.wait(word, parity)) != 0; };
      auto kv_wait = [&](const Cur& c) { return wait_all(&bar->kv_full[c.slot], c.phase); };
      const uint32_t q_lo0 = sw128_desc_lo(q_addr, 16), k_lo0 = sw128_desc_lo(kv_addr, 16), v_lo0 = sw128_desc_lo(kv_addr, PANEL_BYTES);
      auto issue_s = [&](int t, int slot) {               // S_t = Q_t K^T
        const uint32_t qa = q_lo0 + t * (C::TILE_BYTES >> 4), ka = k_lo0 + slot * (C::TILE_BYTES >> 4);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * PANEL_BYTES + (ks & 3) * 32) >> 4;
          umma_f16_ss_parts(tmem_base + t * 128, qa + off, SW128_DESC_HI, ka + off, SW128_DESC_HI, C::IDESC_S, ks != 0 ? 1u : 0u);
        }
      };
      auto issue_pv = [&](int t, int slot, int h64, bool first) {   // O_t += P_t V for the first or second 64 keys
        const uint32_t va = v_lo0 + slot * (C::TILE_BYTES >> 4);
#pragma unroll
        for (int part = 0; part < (HILO ? 2 : 1); ++part)
#pragma unroll
          for (int i = 0; i < 4; ++i) {                   // 16 keys = 8 packed columns of P a step
            const int ks = 4 * h64 + i;
            umma_f16_ts_parts(tmem_base + O_COL + t * D, tmem_base + t * 128 + (ks >> 1) * 32 + (ks & 1) * 8 + part * 16,
                              va + ks * (2048 >> 4), SW128_DESC_HI, C::IDESC_PV, (first && ks == 0 && part == 0) ? 0u : 1u);
          }
      };
      // P of query tile t, tile j of nt, then the next scores into its place
      auto serve = [&](int t, int j, int nt, int before, int items, int v_slot, int k_slot) -> bool {
        if (!wait_all(&bar->p_half[t], uint32_t(before + j) & 1u)) return false;
        if (j == 0 && items > 0 && !wait_all(&bar->o_free[t], uint32_t(items - 1) & 1u)) return false;   // the last output has been read
        tc_fence_after();
        if (elect_one()) issue_pv(t, v_slot, 0, j == 0);
        __syncwarp();
        if (!wait_all(&bar->p_full[t], uint32_t(before + j) & 1u)) return false;
        tc_fence_after();
        if (elect_one()) {
          issue_pv(t, v_slot, 1, false);
          if (j + 1 < nt) { issue_s(t, k_slot); umma_commit(&bar->s_full[t]); }    // behind P V: may overwrite P
          else umma_commit(&bar->o_full[t]);
        }
        __syncwarp();
        return true;
      };
      Work w;
      bool ok = true;
      int k = 0;
      for (; ok && work_at(k, w); ++k) {
        work_done(k);
        const int n0 = w.n0, n1 = w.n1;
        const bool foreign = (w.k0 + n1) * BKEY > w.Lk;   // the last V tile has rows of no key of this sequence
        if ((n0 > 0 && !wait_all(&bar->q_ready[0], uint32_t(items0) & 1u)) || !kv_wait(cur)) { ok = false; break; }
        tc_fence_after();
        if (n0 > 0 && elect_one()) { issue_s(0, cur.slot); umma_commit(&bar->s_full[0]); }
        __syncwarp();
        if (!wait_all(&bar->q_ready[1], uint32_t(k) & 1u)) { ok = false; break; }
        tc_fence_after();
        if (elect_one()) { issue_s(1, cur.slot); umma_commit(&bar->s_full[1]); }
        __syncwarp();
        cur.next();
        for (int j = 0; j < n1 && ok; ++j) {
          const Cur vc = cur;                             // V_j
          cur.next();
          const Cur kc = cur;                             // K_{j+1}
          if (j + 1 < n1) cur.next();
          if (!kv_wait(vc) || (j + 1 < n1 && !kv_wait(kc))) { ok = false; break; }
          if (foreign && j + 1 == n1) {                   // the weights of this step take longer than the clearing
            if (lane == 0) mbar_arrive(&bar->v_here);
            if (!wait_all(&bar->v_clean, uint32_t(cleans) & 1u)) { ok = false; break; }
          }
          if (j < n0 && !serve(0, j, n0, t0, items0, vc.slot, kc.slot)) { ok = false; break; }
          if (!serve(1, j, n1, t1, k, vc.slot, kc.slot)) { ok = false; break; }
        }
        t0 += n0; t1 += n1;
        if (n0 > 0) ++items0;
        if (foreign) ++cleans;
      }
    } else if (warp == 2) {
      // Q scaler: multiplies a landed Q tile by 2^e where it lies
      const __nv_bfloat162 f2 = __float2bfloat162_rn(sc.pow2);
      Work w;
      int items0 = 0;
      bool ok = true;
      for (int k = 0; ok && work_at(k, w); ++k) {
        work_done(k);
        for (int t = 0; t < 2 && ok; ++t) {
          if (t == 0 && w.n0 == 0) continue;
          if (!__all_sync(0xffffffffu, bw.wait(&bar->q_full[t], uint32_t(t == 0 ? items0 : k) & 1u))) { ok = false; break; }
          if (sc.pow2 != 1.0f) {
            uint4* tile = reinterpret_cast<uint4*>(smem + t * C::TILE_BYTES);
#pragma unroll 8
            for (int i = lane; i < C::TILE_BYTES / 16; i += 32) {
              uint4 v = tile[i];
              __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
              h[0] = __hmul2(h[0], f2); h[1] = __hmul2(h[1], f2); h[2] = __hmul2(h[2], f2); h[3] = __hmul2(h[3], f2);
              tile[i] = v;
            }
            fence_async_shared();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->q_ready[t]);
        }
        if (NORMS) {                                      // beside the first products
          for (int t = 0; t < 2 && ok; ++t) {
            if (t == 0 && w.n0 == 0) continue;
            const float norm = largest_row_norm<D>(smem + t * C::TILE_BYTES, lane);
            if (lane == 0) {
              ctl->q_norm[t][(t == 0 ? items0 : k) & 1] = norm;
              mbar_arrive(&bar->q_norm_full[t]);
              mbar_arrive(&bar->q_free[t]);               // with the weight warps' words that the last scores are there
            }
          }
        }
        if (w.n0 > 0) ++items0;
      }
    } else if (warp == 3) {
      // zeroes the rows of a sequence's last V tile that hold none of its keys
      Work w;
      int slot = 0, cleans = 0;                           // ring slot of the item's first tile
      bool ok = true;
      for (int k = 0; ok && work_at(k, w); ++k) {
        work_done(k);
        const int live = max(w.Lk - (w.k0 + w.n1 - 1) * BKEY, 0);
        if (live < BKEY) {
          if (!__all_sync(0xffffffffu, bw.wait(&bar->v_here, uint32_t(cleans) & 1u))) { ok = false; break; }
          unsigned char* tile = smem + C::KV_OFF + (slot + 2 * w.n1 - 1) % C::NKV * C::TILE_BYTES;
          const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
          for (int pn = 0; pn < C::PANELS; ++pn) {
            uint4* panel = reinterpret_cast<uint4*>(tile + pn * PANEL_BYTES);
            for (int i = live * 8 + lane; i < 1024; i += 32) panel[i] = zero;
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->v_clean);
          ++cleans;
        }
        slot = (slot + 2 * w.n1) % C::NKV;
      }
      if (!SECOND && p.zero_tail) {                       // rows of no sequence: before the first, behind the last
        int first, end;
        ragged_extent(p.seqs.cu, p.seqs.S, p.seqs.tokens, first, end);
        const int none = first + p.seqs.tokens - end;
        for (int64_t i = blockIdx.x; i < int64_t(none) * p.H; i += gridDim.x) {
          const int at = int(i / p.H), h = int(i % p.H), row = at < first ? at : end + at - first;
          if (lane < D / 8)
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.o) + row * p.os.t + h * p.os.h + lane * 8) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
    } else {
      const int t = (warp - FIRST_WEIGHT_WARP) >> 2;      // query tile
      const int quarter = warp & 3;
      const int r = quarter * 32 + lane;                  // row of the tile
      const uint32_t lane_sel = uint32_t(quarter * 32) << 16;
      const uint32_t s_taddr = tmem_base + lane_sel + t * 128;
      const uint32_t o_taddr = tmem_base + lane_sel + O_COL + t * D;
      const int tok_r = r / p.G, g_r = r - tok_r * p.G;   // token and head of this row
      // the "scores there" barriers of tile 1, served second in every step, tell that V of the step before and K of this one are read
      const bool releaser = quarter == 0 && lane == 0;
      RingCursor<C::NKV> rel;
      int tiles = 0, items = 0;                           // of this group, in earlier items
      float q_limit = -1.f;                               // queries of smaller squared norm keep every score in the unshifted range
      if (NORMS && p.plan.norms != nullptr) {
        float nk = 0.f;
        for (int i = lane; i < p.plan.norm_ctas; i += 32) nk = max3_abs_nan(nk, p.plan.norms[i], 0.f);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) nk = max3_abs_nan(nk, __shfl_xor_sync(0xffffffffu, nk, o), 0.f);
        // NaN: nothing is below it.  Squares may underflow on one side and overflow on the other: the small term keeps the limit finite, so
        // that an infinite norm is never below it, and no norm is below a limit of zero
        q_limit = sc.y_fast * sc.y_fast / (1.001f * nk + 1e-36f);
      }
      Work w;
      bool ok = true;
      int k = 0;
      for (; ok && work_at(k, w); ++k) {
        const int nk = t == 0 ? w.n0 : w.n1;
        const int tok = (t == 0 ? w.tok0 : w.tok1) + tok_r;
        const bool live = tok_r < TT && tok < w.Lq && (t == 1 || w.has0 != 0);
        const int limit = live ? w.Lk - w.Lq + tok - w.k0 * BKEY : -1;             // last visible key, from the item's first on
        const int limit0 = w.Lk - w.Lq + (t == 0 ? w.tok0 : w.tok1) - w.k0 * BKEY; // of the tile's first row
        const int head = w.head * p.G + g_r;
        float l = 0.f, m_run = 0.f;                       // weights are (rho(x) rho(-m_run) / m)^n: unshifted at first
        const bool whole_sink = live && p.sink != nullptr && w.k0 == 0;
        bool shifted = false, trusted = false;            // the warp's form; its scores need not be looked at
        if (whole_sink) {
          const float b = ragged_sink(p.sink, head, p.inv_c);
          if (!(fabsf(b) <= sc.y_fast * sc.m)) m_run = b;
          l = pow2n_rt(rho_any(b) * (m_run != 0.f ? rho_any(-m_run) : 1.0f) * sc.inv_m, p.log2n);
        }
        shifted = SECOND || __any_sync(0xffffffffu, m_run != 0.f);
        float2 la = make_float2(0.f, 0.f), lb = make_float2(0.f, 0.f);
        for (int j = 0; j < nk && ok; ++j) {
          if (!__all_sync(0xffffffffu, bw.wait(&bar->s_full[t], uint32_t(tiles + j) & 1u))) { ok = false; break; }
          tc_fence_after();
          if (releaser) {
            if (t == 1) {
              if (j > 0) { mbar_arrive(&bar->kv_empty[rel.slot]); rel.next(); }    // V_{j-1}
              mbar_arrive(&bar->kv_empty[rel.slot]); rel.next();                   // K_j
            }
            if (!NORMS && j == nk - 1) mbar_arrive(&bar->q_free[t]);
          }
          const int lim = limit - j * BKEY;
          const bool masked = limit0 - j * BKEY < BKEY - 1;                        // uniform over the group
          if (NORMS && j == 0) {
            if (!__all_sync(0xffffffffu, bw.wait(&bar->q_norm_full[t], uint32_t(items) & 1u))) { ok = false; break; }
            trusted = ctl->q_norm[t][items & 1] < q_limit;
          }
          // Every warp's word that the last scores are there and that it has read the norm: with one warp's word alone the next norm, and the one
          // after, could come while another warp still waits for this one, in an item of one key tile
          if (NORMS && j == nk - 1 && lane == 0) mbar_arrive(&bar->q_free[t]);
          if (!SECOND && !shifted && !trusted) {
            const float sum = tile_square_sum(s_taddr);   // by all lanes: the loads are the whole warp's
            if (!__all_sync(0xffffffffu, !live || sum <= sc.y_fast * sc.y_fast)) {
              const float top = tile_abs_max(s_taddr, lim);
              shifted = __any_sync(0xffffffffu, live && !(top <= sc.y_fast));
            }
          }
          if (!SECOND && !shifted) {
            weigh_tile<LOG2N, HILO>(s_taddr, &bar->p_half[t], &bar->p_full[t], sc.kappa, p.log2n, lim, masked, la, lb);
          } else {
            l += (la.x + la.y) + (lb.x + lb.y);
            la = make_float2(0.f, 0.f); lb = make_float2(0.f, 0.f);
            // the reference moves to the row's largest score so far; with nothing weighed yet it may also fall, to the sink's own where there is
            // one: at zero, weights of 2^-126 and less would be lost beside a sink's of 2^-64
            const float top = tile_row_max(s_taddr, sc.m, lim);
            float m_new = m_run;
            if (lim >= 0 && top > -INFINITY) m_new = j == 0 ? (whole_sink ? fmaxf(ragged_sink(p.sink, head, p.inv_c), top) : top) : l > 0.f ? fmaxf(m_run, top) : top;
            const float alpha = m_new != m_run ? pow2n_rt(rho_any(m_run) * rho_any(-m_new), p.log2n) : 1.0f;
            // O of the earlier tiles is at rest (these scores were issued behind their product): rescale it where a reference moved
            if (__any_sync(0xffffffffu, j > 0 && alpha != 1.0f)) {
              const float a_row = j > 0 ? alpha : 1.0f;
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld_32x32(o_taddr + c, o);
                tmem_ld_wait_for(o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(a_row == 0.f ? 0.f : __uint_as_float(o[i]) * a_row);
                tmem_st_32x32(o_taddr + c, o);
              }
              tmem_st_wait();
            }
            if (l > 0.f) l *= alpha;
            m_run = m_new;
            weigh_tile_shifted<HILO>(s_taddr, &bar->p_half[t], &bar->p_full[t], sc.m, rho_any(-m_run) * sc.inv_m, p.log2n, lim, la, lb);
          }
        }
        if (!ok) break;
        tiles += nk;
        l += (la.x + la.y) + (lb.x + lb.y);
        const bool partial = w.slot >= 0;
        const float inv = l != 0.f ? 1.0f / l : 0.f;      // a row that sees nothing: zero
        const int64_t row = int64_t(w.row0) + tok;
        __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(p.o) + row * p.os.t + head * p.os.h;
        float* dst = nullptr;
        if (partial && (t == 1 || w.has0)) dst = p.plan.slots + ((int64_t(w.slot) * p.Hkv + w.head) * 256 + t * BQ + r) * (D + 4);
        bool write = true;                                // in the second pass: what the first one left infinite or NaN
        if (SECOND) write = live && nk > 0 && (partial ? any_not_finite<D>(dst) : any_not_finite<D>(orow));
        if (dst != nullptr && write) *reinterpret_cast<float4*>(dst + D) = make_float4(nk > 0 && live ? l : 0.f, m_run, 0.f, 0.f);
        if (nk > 0) {
          if (!__all_sync(0xffffffffu, bw.wait(&bar->o_full[t], uint32_t(items) & 1u))) { ok = false; break; }
          ++items;
          if (releaser && t == 1) { mbar_arrive(&bar->kv_empty[rel.slot]); rel.next(); }     // the item's last V tile
          tc_fence_after();
          __nv_bfloat16* lrow = HILO ? static_cast<__nv_bfloat16*>(p.o_lo) + (row * p.H + head) * D : nullptr;
          float most = 0.f;                               // largest number of the row, as it is written
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32(o_taddr + c, o);
            tmem_ld_wait_for(o);
            if (c == D - 32) {                            // O is in registers: the next item may overwrite it
              warp_arrive(&bar->o_free[t]);
            }
            if (!partial) {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(o[i]) * inv);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) most = max3_abs_nan(most, __uint_as_float(o[i]), __uint_as_float(o[i + 1]));
            if (!write) continue;
            if (partial) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<uint4*>(dst + c + 4 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
              continue;
            }
            if (!live) continue;
            uint32_t packed[HILO ? 32 : 16];
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              pack4<HILO>(make_float2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])),
                          make_float2(__uint_as_float(o[i + 2]), __uint_as_float(o[i + 3])), i, packed);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              *reinterpret_cast<uint4*>(orow + c + 8 * i) = make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
              if (HILO) *reinterpret_cast<uint4*>(lrow + c + 8 * i) = make_uint4(packed[16 + 4 * i], packed[17 + 4 * i], packed[18 + 4 * i], packed[19 + 4 * i]);
            }
          }
          // out of range as it is written (a bf16 is infinite from half a step above its largest number on), and not for a NaN among its weights
          if (!SECOND && live && l == l && !(partial ? most <= FLT_LARGEST : most < BF16_INFINITE)) ctl->overflowed[k % RING] = 1;
          // a with p = (rho(x) a)^n: rho(-m_run) (l m^n)^(-1/n)
          if (!partial && live && write && p.stat != nullptr)
            p.stat[int64_t(head) * p.seqs.tokens + row] = l > 0.f ? (m_run != 0.f ? rho_any(-m_run) : 1.0f) * sc.inv_m * inv_root_rt(l, p.log2n) : 0.f;
        }
        work_done(k);
      }
      if (!SECOND) undone = k;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };
  run(std::false_type{});
  if (ctl->abort_flag != 0) {                           // a wait ran out: NaN to the rows that have no result and will get none
    auto spoil = [&](const Work& w) { if (warp >= FIRST_WEIGHT_WARP) spoil_row<D, HILO>(p, w, warp, lane); };
    for (int k = undone; k < ctl->taken; ++k) spoil(ctl->work[k % RING]);
    for (;;) {
      __syncthreads();
      if (threadIdx.x == 0) item_at(int(gridDim.x) + atomicAdd(&p.plan.header->counter, 1), p.plan.header->items * p.Hkv, ctl->work[0]);
      __syncthreads();
      if (ctl->work[0].n1 < 0) break;
      spoil(ctl->work[0]);
    }
  } else if (threadIdx.x == 0) {
    while (ctl->noted < ctl->taken) note();
  }
  if (__syncthreads_or(threadIdx.x == 0 && ctl->abort_flag == 0 && ctl->again >= 0)) run(std::true_type{});

  if (ctl->abort_flag != 0) {
    if (threadIdx.x == 0) {
      if (p.status != nullptr) atomicExch(p.status, ALG_DEV_TIMEOUT);
      const uint64_t t0 = global_timer_ns();            // let issued loads land before shared memory is released
      while (global_timer_ns() - t0 < 200000ull) { }
    }
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Adds up the parts of the items that were cut along the keys: a warp a row, a lane D / 32 columns, references and normalisers one a
// lane, the accumulators of sixteen parts in flight at once.  Parts meet in their order, at the largest of their references, and at 2^-7 of
// their size: 64 finite ones may add up to more than fp32 holds.
template <int D>
__global__ void __launch_bounds__(256) ragged_combine_kernel(const __grid_constant__ RaggedParams p, const ScoreScale sc) {
  griddep_wait();
  constexpr int CPL = D / 32, BATCH = 16;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int units = p.plan.header->combos * p.Hkv * 32;              // eight rows each
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const RaggedCombo it = p.plan.combos[u / (p.Hkv * 32)];
    const int h = (u >> 5) % p.Hkv, in_item = (u & 31) * 8 + warp, t = in_item >> 7, r = in_item & 127;
    const bool two = it.Lq - it.t0 > p.tile_tokens;
    const int tok_r = r / p.G, g = r - tok_r * p.G, tok = it.t0 + (t == 1 && two ? p.tile_tokens : 0) + tok_r;
    if ((t == 0 && !two) || tok_r >= p.tile_tokens || tok >= it.Lq) continue;
    const float* row = p.plan.slots + ((int64_t(it.slot) * p.Hkv + h) * 256 + in_item) * (D + 4);
    const int64_t step = int64_t(p.Hkv) * 256 * (D + 4);            // to the next part
    float m = -INFINITY, l = 0.f, a[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) a[c] = 0.f;
    bool nan = false;
    for (int p0 = 0; p0 < it.parts; p0 += 32) {
      const int n = min(32, it.parts - p0);
      const float2 lm = lane < n ? __ldcg(reinterpret_cast<const float2*>(row + (p0 + lane) * step + D)) : make_float2(0.f, 0.f);
      float f = 0.f;
      for (int b0 = 0; b0 < n; b0 += BATCH) {
        float v[BATCH][CPL];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const float* src = row + (p0 + min(b0 + j, n - 1)) * step + lane * CPL;
          if (CPL == 4) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
            v[j][0] = x.x; v[j][1] = x.y; v[j][CPL - 2] = x.z; v[j][CPL - 1] = x.w;
          } else {
            const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
            v[j][0] = x.x; v[j][1] = x.y;
          }
        }
        if (b0 == 0) {                                 // a part that weighed nothing has no say in the reference
          nan |= __any_sync(0xffffffffu, lm.x != lm.x) != 0;
          const float top = fmaxf(m, warp_max(lm.x > 0.f ? lm.y : -INFINITY));
          if (top > m) {
            const float old = m > -INFINITY ? pow2n_rt(rho_any(m) * rho_any(-top), p.log2n) : 0.f;
            l *= old;
#pragma unroll
            for (int c = 0; c < CPL; ++c) a[c] *= old;
            m = top;
          }
          f = lm.x > 0.f ? (lm.y == m ? 1.0f : pow2n_rt(rho_any(lm.y) * rho_any(-m), p.log2n)) : 0.f;
          l += warp_sum(f * lm.x);
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const float fj = __shfl_sync(0xffffffffu, f, (b0 + j) & 31) * 0x1p-7f;
          if (b0 + j < n && fj != 0.f) {               // else the accumulator may never have been written
#pragma unroll
            for (int c = 0; c < CPL; ++c) a[c] = fmaf(fj, v[j][c], a[c]);
          }
        }
      }
    }
    const float inv = nan ? __int_as_float(0x7fc00000) : l > 0.f ? 1.0f / l : 0.f;
    const int64_t at = int64_t(it.row0) + tok;
    const int head = h * p.G + g;
    __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(p.o) + at * p.os.t + head * p.os.h + lane * CPL;
    __nv_bfloat16* lrow = p.o_lo != nullptr ? static_cast<__nv_bfloat16*>(p.o_lo) + (at * p.H + head) * D + lane * CPL : nullptr;
#pragma unroll
    for (int c = 0; c < CPL; c += 2) {
      const float x = a[c] * inv * 0x1p7f, y = a[c + 1] * inv * 0x1p7f;
      const uint32_t hi = pack_bf16(x, y);
      *reinterpret_cast<uint32_t*>(orow + c) = hi;
      if (lrow != nullptr) *reinterpret_cast<uint32_t*>(lrow + c) = pack_bf16(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
    }
    if (p.stat != nullptr && lane == 0) {
      const float stat = l > 0.f ? rho_any(-m) * sc.inv_m * inv_root_rt(l, p.log2n) : 0.f;
      p.stat[int64_t(head) * p.seqs.tokens + at] = nan ? __int_as_float(0x7fc00000) : stat;
    }
  }
}

template <int D, int LOG2N, bool HILO, bool PAGED>
int launch_kernel(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const RaggedParams& p, const ScoreScale& sc, int grid,
                  cudaStream_t stream) {
  auto kern = ragged_attn_kernel<D, LOG2N, HILO, PAGED>;
  static PerDeviceOnce configured;
  if (int rc = configured.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem_bytes<D>())); })) return rc;
  ALG_CUDA_TRY(launch_dependent(kern, dim3(grid), dim3(NTHREADS), smem_bytes<D>(), stream, tq, tk, tv, p, sc));
  count_launch();
  return ALG_OK;
}

template <int D>
int launch_d(const RaggedParams& p, cudaStream_t stream) {
  CUtensorMap tq, tk, tv;
  const uint64_t tokens = uint64_t(p.seqs.tokens);
  {
    const uint64_t dims[4] = {64, uint64_t(p.H), tokens, uint64_t(D / 64)};
    const uint64_t strides[3] = {uint64_t(p.qs.h), uint64_t(p.qs.t), 64};
    const uint32_t box[4] = {64, uint32_t(p.G), uint32_t(p.tile_tokens), 1};
    if (int rc = make_tmap_bf16(&tq, p.q, 4, dims, strides, box, true)) return rc;
  }
  for (int i = 0; i < 2; ++i) {
    const Strides2& s = i == 0 ? p.ks : p.vs;
    const void* base = i == 0 ? p.k : p.v;
    CUtensorMap* tm = i == 0 ? &tk : &tv;
    if (p.table != nullptr) {
      const uint64_t dims[5] = {64, uint64_t(p.page), uint64_t(D / 64), uint64_t(p.Hkv), uint64_t(p.pages)};
      const uint64_t strides[4] = {uint64_t(s.t), 64, uint64_t(s.h), uint64_t(i == 0 ? p.k_page : p.v_page)};
      const uint32_t box[5] = {64, uint32_t(std::min(p.page, BKEY)), 1, 1, 1};
      if (int rc = make_tmap_bf16(tm, base, 5, dims, strides, box, true)) return rc;
    } else {
      const uint64_t dims[4] = {64, tokens, uint64_t(D / 64), uint64_t(p.Hkv)};
      const uint64_t strides[3] = {uint64_t(s.t), 64, uint64_t(s.h)};
      const uint32_t box[4] = {64, uint32_t(BKEY), uint32_t(D / 64), 1};
      if (int rc = make_tmap_bf16(tm, base, 4, dims, strides, box, true)) return rc;
    }
  }
  ScoreScale sc;
  {
    int ex = 0;
    const double f = frexp(double(p.scale), &ex);         // scale = f 2^ex = 2^(ex - 1) m, 1 <= m < 2
    const double m = 2.0 * f;
    sc.pow2 = float(ldexp(1.0, ex - 1));
    sc.m = float(m); sc.inv_m = float(1.0 / m); sc.kappa = float(1.0 / (m * m));
    sc.y_fast = float(ragged_fast_range(1 << p.log2n) / m);
  }
  const int64_t most = int64_t(p.plan.max_items) * p.Hkv;
  const int grid = int(std::min<int64_t>(most, p.plan.sms));
  const bool hilo = p.o_lo != nullptr, paged = p.table != nullptr;
  int rc;
  if (p.log2n == 4) {
    if (paged) rc = launch_kernel<D, 4, false, true>(tq, tk, tv, p, sc, grid, stream);
    else if (hilo) rc = launch_kernel<D, 4, true, false>(tq, tk, tv, p, sc, grid, stream);
    else rc = launch_kernel<D, 4, false, false>(tq, tk, tv, p, sc, grid, stream);
  } else {
    if (paged) rc = launch_kernel<D, 0, false, true>(tq, tk, tv, p, sc, grid, stream);
    else if (hilo) rc = launch_kernel<D, 0, true, false>(tq, tk, tv, p, sc, grid, stream);
    else rc = launch_kernel<D, 0, false, false>(tq, tk, tv, p, sc, grid, stream);
  }
  if (rc) return rc;
  if (p.plan.max_slots > 0) {
    const int blocks = int(std::min<int64_t>(int64_t(p.plan.max_combos) * p.Hkv * 32, int64_t(p.plan.sms) * 8));
    ALG_CUDA_TRY(launch_dependent(ragged_combine_kernel<D>, dim3(std::max(blocks, 1)), dim3(256), 0, stream, p, sc));
    count_launch();
  }
  return ALG_OK;
}

}  // namespace

int launch_ragged_attention(const RaggedParams& p, cudaStream_t stream) {
  if (int rc = launch_ragged_plan(p, stream)) return rc;
  return p.D == 64 ? launch_d<64>(p, stream) : launch_d<128>(p, stream);
}

}  // namespace alg
