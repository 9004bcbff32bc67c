// Backward of the attention over packed sequences with grouped heads: tcgen05.
//
//   p_ij = (rho(x_ij) a_i)^n from the saved statistic, dP = dO V^T, delta_i = dO_i . o_i
//   dS = n p (dP - delta) / sqrt(1 + x^2) / (sqrt(D) c),  dQ = dS K,  dK = sum over the group of dS^T Q,  dV = sum of P^T dO
//   dsink_h = - n / c / sqrt(1 + (b/c)^2) sum_i p_sink,i delta_i
//
// The two kinds of CTA, the tensor-memory layout and the two element-wise phases of a step are those of attn_bwd_sm100.cu (MODE 0:
// rows are queries, dQ; MODE 1: rows are keys, dK and dV).  What is different:
//   - blocks come from a list per kind, longest first, that a plan kernel makes of the lengths on the device; a CTA whose number is
//     behind the list's end leaves at once;
//   - MODE 1 streams the queries of all heads of the group, one head behind the other, into one pair of accumulators: the sum over the
//     group is formed in fp32 and written once, in an order that does not change;
//   - tiles read on into the next sequence.  Its rows are masked or have statistic 0, but 0 times a NaN or infinity is NaN, so
//     the producer warp zeroes the foreign rows of a streamed tile before the tensor core reads it;
//   - any scores: 16 columns at a time go the short way, y + sqrt(kappa + y^2), where all their |x| of the warp's rows are within
//     the range of the forward's unshifted weights, else the cancellation-free one;
//   - delta takes the forward's output as two bf16 halves.  dsink is a float32 sum over all tokens, for which the 16 bits of these, and of
//     the weights that made them, are still too coarse (2 to 3e-6 of it): the query blocks add up delta_i = sum_j p_ij dP_ij
//     and l_i = p_sink,i + sum_j p_ij from the weights in fp32, a row's share is p_sink delta / l^2 (l is 1 but for the statistic's last bits),
//     and blocks' shares are added in a fixed order by the block that arrives last.
// Bound as the batched backward is: the element-wise phases, a tensor-memory load and an mbarrier between every two products.  Measured
// with the forward (sequences of 2314, 2770 and 4096, 16 heads of 128): 830 us, 515 TFLOP/s of 3.5 times the forward's products, the
// forward's second half of the weights not counted; of it 5 % are the sinks' sums.  20 sequences of 72 to 1024, 12 heads on 4 of 64: the GPU's
// part is 140 us, the call's 176 to 182 (autograd's host side).
#include "common.cuh"
#include "ragged.cuh"
#include "sm100_ptx.cuh"

#include <type_traits>

namespace alg {
namespace {

using namespace sm100;

constexpr int BT = 128;                          // resident rows of a CTA
constexpr int RES_PANEL = BT * 128;              // one 64-column panel of a resident tile
constexpr int MAX_STEPS = 4;

template <int D, int BS, int CTAS> struct Cfg {
  static constexpr int PANELS = D / 64;
  static constexpr int RES_BYTES = PANELS * RES_PANEL;
  static constexpr int STR_PANEL = BS * 128, STR_BYTES = PANELS * STR_PANEL;
  static constexpr int NS = (D == 128) ? 2 : 4;                 // ring depth in steps (two streamed tiles per step)
  static constexpr int NG = BS / 32;                            // column groups of the element-wise stage
  static constexpr int EW_WARPS = 4 * NG, NTHREADS = 64 + 32 * EW_WARPS;
  static constexpr int RING_OFF = 2 * RES_BYTES;
  static constexpr int VEC_OFF = RING_OFF + NS * 2 * STR_BYTES; // MODE 1: per ring slot BS statistics, BS negated deltas
  static constexpr int CTL_OFF = VEC_OFF + NS * 2 * BS * 4;
  static constexpr uint32_t TMEM_COLS = 512 / CTAS;
  static constexpr uint32_t S_COL = 0, DP_COL = BS, ACC0_COL = 2 * BS, ACC1_COL = 2 * BS + D;
  static constexpr uint32_t s1_col(int mode) { return 2 * BS + (mode + 1) * D; }
  // a second S buffer where tensor memory has room for it: S of step j + 1 is then computed while the threads
  // are still reading S of step j
  static constexpr bool double_s(int mode) { return s1_col(mode) + BS <= TMEM_COLS; }
  static constexpr uint32_t IDESC_S = make_idesc_bf16(BT, BS, 0, 0);
  static constexpr uint32_t IDESC_TS = make_idesc_bf16(BT, D, 0, 1);
};

struct __align__(16) Control {
  uint64_t clean[MAX_STEPS];      // the slot's foreign rows are zeroed
  uint64_t never;                 // at which nothing arrives
  uint64_t res_full, full[MAX_STEPS], empty[MAX_STEPS], vec_full[MAX_STEPS], s_full[2], dp_full, p_done[2], ds_done, acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

// has the phase completed? (does not wait)
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}

template <class C> constexpr size_t smem_bytes() { return size_t(C::CTL_OFF) + sizeof(Control) + 1024; }

// 16 scores y of this thread's row -> the weights p (packed bf16 pairs in pw) and the factor scale p / sqrt(1 + x^2) that phase 2
// multiplies (dP - delta) by, x = scale y, kappa = 1 / scale^2.  `a2`: scale times the statistic, by row (MODE 0: a2[0]) or by
// column (MODE 1: a2[0..7]).
//   short:  scale (y + sqrt(kappa + y^2)) = rho(x),  rsqrt(kappa + y^2) = scale / sqrt(1 + x^2)
// `pw`: the weights, as bf16 pairs (MODE 1) or, where the sinks' gradients need them, in fp32 (MODE 0).
template <bool BY_COLUMN, bool SINK, int LOG2N, bool MASK>
__device__ __forceinline__ void weights16(const uint32_t* s, float2* slope, uint32_t* pw, const float2* a2, float scale, float kappa,
                                          float y_fast, int log2n, int row, int col0, bool live) {
  const float2 kp = make_float2(kappa, kappa);
  float2 t[8];
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max3_abs_nan(most, __uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
  if (!__any_sync(0xffffffffu, live && !(most <= y_fast))) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 y = make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), rad = __ffma2_rn(y, y, kp);
      slope[i] = make_float2(rsqrt_approx(rad.x), rsqrt_approx(rad.y));
      t[i] = __fmul2_rn(__ffma2_rn(rad, slope[i], y), BY_COLUMN ? a2[i] : a2[0]);
    }
  } else {
    const float inv_scale = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = __uint_as_float(s[2 * i]) * scale, y = __uint_as_float(s[2 * i + 1]) * scale;
      const float2 a = BY_COLUMN ? a2[i] : a2[0];
      slope[i] = make_float2(scale * rsqrt_approx(fmaf(x, x, 1.0f)), scale * rsqrt_approx(fmaf(y, y, 1.0f)));
      t[i] = make_float2(rho_any(x) * (a.x * inv_scale), rho_any(y) * (a.y * inv_scale));
    }
  }
  // the power as passes over the eight pairs, so that every pass has independent multiplications
  if (LOG2N > 0) {
#pragma unroll
    for (int it = 0; it < LOG2N; ++it)
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = __fmul2_rn(t[i], t[i]);
  } else {
    for (int it = 0; it < log2n; ++it)
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = __fmul2_rn(t[i], t[i]);
  }
  if (MASK) {   // causal, key <= query: rows are keys where the factors come by column, else queries
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col0 + 2 * i;
      if (BY_COLUMN ? (c < row) : (c > row)) t[i].x = 0.f;
      if (BY_COLUMN ? (c + 1 < row) : (c + 1 > row)) t[i].y = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    slope[i] = __fmul2_rn(slope[i], t[i]);
    if (BY_COLUMN) {
      pw[i] = pack_bf16(t[i].x, t[i].y);
    } else if (SINK) {
      pw[2 * i] = __float_as_uint(t[i].x);
      pw[2 * i + 1] = __float_as_uint(t[i].y);
    }
  }
}

// Phase 1 on this thread's 32 scores at tensor-memory address s_t; `vec`: the columns' statistics in shared memory
// (MODE 1).  MODE 1 leaves the packed weights over the columns read, SINK the weights in fp32 over the scores.
template <int MODE, bool SINK, int LOG2N, bool MASK>
__device__ __forceinline__ void phase1(uint32_t s_t, float2* slope, const float* vec, float2 a_row, float scale, float kappa, float y_fast,
                                       int log2n, int row, int col0, bool live) {
  uint32_t s0[16], s1[16];
  tmem_ld_32x16(s_t, s0);
  tmem_ld_wait_for16(s0);
  tmem_ld_32x16(s_t + 16, s1);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t pw[16];
    float2 a2[8];
    if (MODE == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(vec + c * 16 + 4 * i);
        a2[2 * i] = make_float2(v.x, v.y);
        a2[2 * i + 1] = make_float2(v.z, v.w);
      }
    } else {
      a2[0] = a_row;
    }
    if (c == 1) tmem_ld_wait_for16(s1);
    weights16<MODE == 1, SINK, LOG2N, MASK>(c == 0 ? s0 : s1, slope + 8 * c, pw, a2, scale, kappa, y_fast, log2n, row, col0 + c * 16, live);
    if (MODE == 1) tmem_st_32x8(s_t + c * 8, pw);
    if (SINK) tmem_st_32x16(s_t + c * 16, pw);
  }
}

template <class C, int D, int BS, int MODE>
__device__ __forceinline__ void bwd_block(unsigned char* smem, Control* ctl, const CUtensorMap* tm_q, const CUtensorMap* tm_k,
                                          const CUtensorMap* tm_v, const CUtensorMap* tm_do, const RaggedBwdParams& p, const int4& block, int h) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tmem_base = ctl->tmem_base;
  const BoundedWait bw{&ctl->abort_flag, 1000000000ull};
  constexpr bool DB = C::double_s(MODE);
  auto sbuf = [](int j) { return DB ? (j & 1) : 0; };
  auto sphase = [](int j) -> uint32_t { return DB ? ((j >> 1) & 1u) : (j & 1u); };
  auto s_col = [](int j) -> uint32_t { return (DB && (j & 1)) ? C::s1_col(MODE) : C::S_COL; };

  // h: query head (MODE 0) or key head (MODE 1); rows are counted in the sequence, which lies at packed row `base`
  const int base = block.x, L = block.y, row0 = block.z;
  const int first = (MODE == 0) ? 0 : row0;                  // first streamed row
  const int end = (MODE == 0) ? min(row0 + BT, L) : L;       // one past the last
  const int nq = (end - first + BS - 1) / BS;                // steps of a head
  const int nsteps = (MODE == 0) ? nq : nq * p.G;
  const bool foreign = first + nq * BS > L;                  // a head's last tiles read on into the next sequence
  const int kv_head = (MODE == 0) ? h / p.G : h;

  if (warp == 0) {
    const CUtensorMap* res0 = (MODE == 0) ? tm_q : tm_k;     // A operand of the first score product
    const CUtensorMap* res1 = (MODE == 0) ? tm_do : tm_v;    // A operand of the second
    const CUtensorMap* str0 = (MODE == 0) ? tm_k : tm_q;     // their streamed B operands
    const CUtensorMap* str1 = (MODE == 0) ? tm_v : tm_do;
    if (lane == 0) {
      mbar_arrive_expect_tx(&ctl->res_full, 2 * C::RES_BYTES);
      for (int r = 0; r < BT; r += BS) {                     // boxes are BS rows high, all panels
        tma_load_4d(smem + r * 128, res0, &ctl->res_full, 0, base + row0 + r, 0, h);
        tma_load_4d(smem + C::RES_BYTES + r * 128, res1, &ctl->res_full, 0, base + row0 + r, 0, h);
      }
    }
    // MODE 1: statistic (times the score scale) and delta of the next step's queries, fetched one step ahead
    constexpr int VPL = BS / 32;
    float st[VPL], dl[VPL];
    auto fetch = [&](int g, int j) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int t = first + j * BS + i * 32 + lane;
        const bool in = t < L;
        const int64_t at = int64_t(h * p.G + g) * p.tokens + base + t;
        st[i] = in ? __ldg(p.stat + at) * p.scale : 0.f;
        dl[i] = in ? __ldg(p.delta + at) : 0.f;
      }
    };
    // zeroes the rows of a head's last tiles that are not this sequence's, once they have landed
    auto clear = [&](int j) -> bool {
      const int slot = j % C::NS;
      if (__any_sync(0xffffffffu, !bw.wait(&ctl->full[slot], (j / C::NS) & 1u))) return false;
      const int keep = L - (first + (nq - 1) * BS);
      unsigned char* dst = smem + C::RING_OFF + slot * 2 * C::STR_BYTES;
      for (int pn = 0; pn < 2 * C::PANELS; ++pn) {
        uint4* panel = reinterpret_cast<uint4*>(dst + pn * C::STR_PANEL);
        for (int i = keep * 8 + lane; i < BS * 8; i += 32) panel[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->clean[slot]);
      return true;
    };
    if (MODE == 1) fetch(0, 0);
    bool ok = true;
    int g = 0, jq = 0;                                       // head of the group, step of the head
    const int loads = min(nsteps, p.limits.max_loads);
    for (int j = 0; j < loads; ++j) {
      const int slot = j % C::NS;
      // The clearing of a head's last tiles comes behind the next step's loads, which then do not wait for the landing; but where the
      // slot for these is not free yet it comes first: what frees the slot may be waiting for the cleared tiles.
      bool to_clear = foreign && jq == 0 && j > 0;
      if (to_clear && !__all_sync(0xffffffffu, mbar_test(&ctl->empty[slot], ((j / C::NS) & 1u) ^ 1u))) {
        if (!clear(j - 1)) { ok = false; break; }
        to_clear = false;
      }
      if (__any_sync(0xffffffffu, !bw.wait(&ctl->empty[slot], ((j / C::NS) & 1u) ^ 1u))) { ok = false; break; }
      if (lane == 0) {
        unsigned char* dst = smem + C::RING_OFF + slot * 2 * C::STR_BYTES;
        mbar_arrive_expect_tx(&ctl->full[slot], 2 * C::STR_BYTES);
        const int head = (MODE == 0) ? kv_head : h * p.G + g;
        tma_load_4d(dst, str0, &ctl->full[slot], 0, base + first + jq * BS, 0, head);
        tma_load_4d(dst + C::STR_BYTES, str1, &ctl->full[slot], 0, base + first + jq * BS, 0, head);
      }
      if (++jq == nq) { jq = 0; ++g; }
      if (MODE == 1) {
        float* vec = reinterpret_cast<float*>(smem + C::VEC_OFF) + slot * 2 * BS;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
          vec[i * 32 + lane] = st[i];
          vec[BS + i * 32 + lane] = -dl[i];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->vec_full[slot]);
        if (j + 1 < nsteps) fetch(g, jq);
      }
      __syncwarp();
      if (to_clear && !clear(j - 1)) { ok = false; break; }
    }
    if (loads < nsteps) BoundedWait{&ctl->abort_flag, p.limits.budget_ns}.wait(&ctl->never, 0);     // in vain
    else if (ok && foreign) clear(nsteps - 1);
  } else if (warp == 1) {
    // the whole warp runs the loop and one elected lane issues (cheaper per issue than a lane-0 branch)
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, bw.wait(bar, parity)) != 0; };
    const uint32_t res_addr = smem_u32(smem), ring_addr = smem_u32(smem + C::RING_OFF);
    const uint32_t a0_lo = sw128_desc_lo(res_addr, 16), a1_lo = sw128_desc_lo(res_addr + C::RES_BYTES, 16);
    // S-like product: d = A . B^T, both K-major tiles of D columns
    auto issue_scores = [&](uint32_t d_tmem, uint32_t a_lo, uint32_t b_addr) {
      const uint32_t b_lo = sw128_desc_lo(b_addr, 16);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint32_t a_off = ((ks >> 2) * RES_PANEL + (ks & 3) * 32) >> 4, b_off = ((ks >> 2) * C::STR_PANEL + (ks & 3) * 32) >> 4;
        umma_f16_ss_parts(d_tmem, a_lo + a_off, SW128_DESC_HI, b_lo + b_off, SW128_DESC_HI, C::IDESC_S, ks != 0 ? 1u : 0u);
      }
    };
    // acc += W . B: W = packed bf16 in tensor memory (see the head of the file), B = a streamed [row][D] tile read
    // as an MN-major operand
    auto issue_product = [&](uint32_t d_tmem, uint32_t w_tmem, uint32_t b_addr, bool first_step) {
      const uint32_t b_lo = sw128_desc_lo(b_addr, C::STR_PANEL);
#pragma unroll
      for (int ks = 0; ks < BS / 16; ++ks)
        umma_f16_ts_parts(d_tmem, w_tmem + (ks >> 1) * 32 + (ks & 1) * 8, b_lo + ks * (2048 >> 4), SW128_DESC_HI, C::IDESC_TS,
                          (first_step && ks == 0) ? 0u : 1u);
    };
    auto tile0 = [&](int j) { return ring_addr + (j % C::NS) * 2 * C::STR_BYTES; };
    uint32_t cleaned = 0;                                    // per slot: parity of how often it was cleared
    int at_head = 0;                                         // step of the head that comes next
    auto score_s = [&](int j) -> bool {                      // waits for step j's tiles, then S (or S^T) of step j
      const int slot = j % C::NS;
      if (!wait_all(&ctl->full[slot], (j / C::NS) & 1u)) return false;
      if (++at_head == nq) {
        at_head = 0;
        if (foreign) {
          if (!wait_all(&ctl->clean[slot], (cleaned >> slot) & 1u)) return false;
          cleaned ^= 1u << slot;
        }
      }
      tc_fence_after();
      if (elect_one()) {
        issue_scores(tmem_base + s_col(j), a0_lo, tile0(j));
        umma_commit(&ctl->s_full[sbuf(j)]);
      }
      __syncwarp();
      return true;
    };
    auto score_dp = [&](int j) {                             // dP (or dP^T) of step j, whose tiles score_s(j) has waited for
      if (elect_one()) {
        issue_scores(tmem_base + C::DP_COL, a1_lo, tile0(j) + C::STR_BYTES);
        umma_commit(&ctl->dp_full);
      }
      __syncwarp();
    };
    bool ok = wait_all(&ctl->res_full, 0) && score_s(0);
    if (ok) {
      score_dp(0);
      if (DB && nsteps > 1) ok = score_s(1);
    }
    for (int j = 0; j < nsteps && ok; ++j) {
      const bool has_next = j + 1 < nsteps;
      const uint32_t t0 = tile0(j), t1 = t0 + C::STR_BYTES;
      // phase 1 is over: S has been read (MODE 1: P^T stands in its place)
      if (!wait_all(&ctl->p_done[sbuf(j)], sphase(j))) { ok = false; break; }
      tc_fence_after();
      if (MODE == 1) {
        if (elect_one()) issue_product(tmem_base + C::ACC0_COL, tmem_base + s_col(j), t1, j == 0);     // dV += P^T dO
        __syncwarp();
      }
      if (!DB && has_next && !score_s(j + 1)) { ok = false; break; }     // after the dV product: may overwrite P^T
      // phase 2 is over: dS stands in place of dP
      if (!wait_all(&ctl->ds_done, j & 1u)) { ok = false; break; }
      tc_fence_after();
      if (elect_one()) {
        issue_product(tmem_base + (MODE == 0 ? C::ACC0_COL : C::ACC1_COL), tmem_base + C::DP_COL, t0, j == 0);   // dQ += dS K / dK += dS^T Q
        umma_commit(&ctl->empty[j % C::NS]);
      }
      __syncwarp();
      if (has_next) score_dp(j + 1);                         // after that product: may overwrite dS
      if (DB && j + 2 < nsteps && !score_s(j + 2)) { ok = false; break; }   // into the buffer phase 1 of step j has left
    }
    if (ok && elect_one()) umma_commit(&ctl->acc_full);
  } else {
    const int quarter = warp & 3, group = (warp - 2) >> 2;
    const int r = quarter * 32 + lane, row = row0 + r;
    const int wrow0 = row0 + quarter * 32;                    // this warp's first row
    const uint32_t lane_sel = uint32_t(quarter * 32) << 16;
    const float kappa = 1.0f / (p.scale * p.scale);
    const bool live = row < L;
    float2 a_row = make_float2(0.f, 0.f), delta_row = make_float2(0.f, 0.f);
    if (MODE == 0 && live) {
      const int64_t at = int64_t(h) * p.tokens + base + row;
      const float a = p.stat[at] * p.scale, d = -p.delta[at];
      a_row = make_float2(a, a);
      delta_row = make_float2(d, d);
    }
    const uint32_t dp_t = tmem_base + lane_sel + C::DP_COL + group * 32;
    float row_delta = 0.f, row_sum = 0.f;                     // of this thread's columns
    auto steps = [&](auto power, auto sunk) -> bool {
      constexpr int LOG2N = decltype(power)::value;
      constexpr bool SINK = MODE == 0 && decltype(sunk)::value;
      static_assert(!SINK || DB, "the weights stay where the scores were until phase 2 has read them");
      int slot = 0;
      uint32_t ring = 0;                                      // ring position and phase
      for (int j = 0; j < nsteps; ++j) {
        const int col0 = first + (MODE == 0 ? j : j % nq) * BS + group * 32;     // first streamed row of this thread's 32 columns
        const float* vec = reinterpret_cast<const float*>(smem + C::VEC_OFF) + slot * 2 * BS + group * 32;
        float2 slope[16];
        // ---- phase 1: scores -> weights
        const uint32_t s_t = tmem_base + lane_sel + s_col(j) + group * 32;
        if (MODE == 1 && !bw.wait(&ctl->vec_full[slot], ring)) return false;
        if (++slot == C::NS) { slot = 0; ring ^= 1u; }
        if (!bw.wait(&ctl->s_full[sbuf(j)], sphase(j))) return false;
        tc_fence_after();
        // the causal mask removes none, some or all of a 32 x 32 block (warp-uniform)
        const int ahead = (MODE == 0) ? col0 - wrow0 : wrow0 - col0;      // > -32: some, >= 32: all
        if (ahead <= -32) {
          phase1<MODE, SINK, LOG2N, false>(s_t, slope, vec, a_row, p.scale, kappa, p.y_fast, p.log2n, row, col0, live);
        } else if (ahead < 32) {
          phase1<MODE, SINK, LOG2N, true>(s_t, slope, vec, a_row, p.scale, kappa, p.y_fast, p.log2n, row, col0, live);
        } else {
          uint32_t zero[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) { slope[i] = make_float2(0.f, 0.f); zero[i] = 0u; }
          if (MODE == 1) tmem_st_32x16(s_t, zero);
        }
        if (MODE == 1) tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->p_done[sbuf(j)]);
        // ---- phase 2: dP -> dS = slope (dP - delta)
        if (!bw.wait(&ctl->dp_full, j & 1u)) return false;
        tc_fence_after();
        uint32_t d0[16], d1[16], w[16];
        // sums of sixteen columns at a time: a long row's sum is one of short sums
        auto add_row = [&](const uint32_t* dp) {
          float2 ds2 = make_float2(0.f, 0.f), l2 = ds2;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 wv = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
            ds2 = __ffma2_rn(wv, make_float2(__uint_as_float(dp[2 * i]), __uint_as_float(dp[2 * i + 1])), ds2);
            l2 = __fadd2_rn(l2, wv);
          }
          row_delta += ds2.x + ds2.y;
          row_sum += l2.x + l2.y;
        };
        tmem_ld_32x16(dp_t, d0);
        if (SINK && ahead < 32) {
          tmem_st_wait();                                     // phase 1's
          tmem_ld_32x16(s_t, w);
          tmem_ld_wait_for16(w);
          tmem_ld_wait_for16(d0);
          add_row(d0);
        } else {
          tmem_ld_wait_for16(d0);
        }
        tmem_ld_32x16(dp_t + 16, d1);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float2 nd[8];
          if (MODE == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 v = *reinterpret_cast<const float4*>(vec + BS + c * 16 + 4 * i);
              nd[2 * i] = make_float2(v.x, v.y);
              nd[2 * i + 1] = make_float2(v.z, v.w);
            }
          }
          if (c == 1) {
            if (SINK && ahead < 32) {
              tmem_ld_32x16(s_t + 16, w);
              tmem_ld_wait_for16(w);
            }
            tmem_ld_wait_for16(d1);
            if (SINK && ahead < 32) add_row(d1);
          }
          const uint32_t* dp = c == 0 ? d0 : d1;
          uint32_t ds[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 d = make_float2(__uint_as_float(dp[2 * i]), __uint_as_float(dp[2 * i + 1]));
            const float2 v = __fmul2_rn(slope[8 * c + i], __fadd2_rn(d, MODE == 1 ? nd[i] : delta_row));
            ds[i] = pack_bf16(v.x, v.y);
          }
          tmem_st_32x8(dp_t + c * 8, ds);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->ds_done);
      }
      return true;
    };
    using std::integral_constant;
    const bool sunk = MODE == 0 && p.dsink != nullptr;
    const bool ok = p.log2n == 4 ? (sunk ? steps(integral_constant<int, 4>{}, std::true_type{}) : steps(integral_constant<int, 4>{}, std::false_type{}))
                                 : (sunk ? steps(integral_constant<int, 0>{}, std::true_type{}) : steps(integral_constant<int, 0>{}, std::false_type{}));
    if (ok && bw.wait(&ctl->acc_full, 0)) {
      tc_fence_after();
      if (sunk)                                                // the ring has been read to its end
        reinterpret_cast<float2*>(smem + C::RING_OFF)[group * BT + r] = live ? make_float2(row_delta, row_sum) : make_float2(0.f, 0.f);
      constexpr int CPT = D / C::NG;                           // accumulator columns per thread
      const int64_t at = int64_t(base) + row;
      __nv_bfloat16* out0 = ((MODE == 0) ? p.dq + at * p.dqs.t + h * p.dqs.h : p.dv + at * p.dvs.t + h * p.dvs.h) + group * CPT;
      __nv_bfloat16* out1 = (MODE == 1) ? p.dk + at * p.dks.t + h * p.dks.h + group * CPT : nullptr;
      const float n_fac = p.n_f;                                // the factor the element-wise stage left out; dV carries none
#pragma unroll 1
      for (int which = 0; which < (MODE == 0 ? 1 : 2); ++which) {
        const uint32_t acc_t = tmem_base + lane_sel + (which == 0 ? C::ACC0_COL : C::ACC1_COL) + group * CPT;
        __nv_bfloat16* dst = which == 0 ? out0 : out1;
        const float fac = (MODE == 0 || which == 1) ? n_fac : 1.0f;
#pragma unroll 1
        for (int c = 0; c < CPT / 16; ++c) {
          uint32_t a[16];
          tmem_ld_32x16(acc_t + c * 16, a);
          tmem_ld_wait_for16(a);
          if (live) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              *reinterpret_cast<uint4*>(dst + c * 16 + i * 8) =
                  make_uint4(pack_bf16(__uint_as_float(a[8 * i]) * fac, __uint_as_float(a[8 * i + 1]) * fac),
                             pack_bf16(__uint_as_float(a[8 * i + 2]) * fac, __uint_as_float(a[8 * i + 3]) * fac),
                             pack_bf16(__uint_as_float(a[8 * i + 4]) * fac, __uint_as_float(a[8 * i + 5]) * fac),
                             pack_bf16(__uint_as_float(a[8 * i + 6]) * fac, __uint_as_float(a[8 * i + 7]) * fac));
          }
        }
      }
    }
  }
}

// A wait ran out: NaN to the block's rows, whatever they hold.
template <int D>
__device__ __forceinline__ void spoil_block(const RaggedBwdParams& p, const int4& block, int h, bool keys) {
  const uint4 nan = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
#pragma unroll 1
  for (int i = threadIdx.x; i < BT * (D / 8); i += blockDim.x) {
    const int row = block.z + i / (D / 8), col = i % (D / 8) * 8;
    if (row >= block.y) continue;
    const int64_t at = int64_t(block.x) + row;
    *reinterpret_cast<uint4*>((keys ? p.dv + at * p.dvs.t + h * p.dvs.h : p.dq + at * p.dqs.t + h * p.dqs.h) + col) = nan;
    if (keys) *reinterpret_cast<uint4*>(p.dk + at * p.dks.t + h * p.dks.h + col) = nan;
  }
}

// A query block's share of dsink, from the rows' sums that its threads left in shared memory; the block that arrives last adds up all
// shares, in the order of the blocks in the call.  The power of the sink's weight is taken in 64 bits, of the statistic as the weights had it.
template <class C>
__device__ void sink_share(unsigned char* smem, const Control* ctl, const RaggedBwdParams& p, const int4& block, int h, int n) {
  float* scratch = reinterpret_cast<float*>(smem);             // the resident tiles have been read
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < BT) {
    float share = 0.f;
    if (block.z + int(threadIdx.x) < block.y) {
      float delta = 0.f, l = 0.f;
#pragma unroll
      for (int g = 0; g < C::NG; ++g) {
        const float2 v = reinterpret_cast<const float2*>(smem + C::RING_OFF)[g * BT + threadIdx.x];
        delta += v.x;
        l += v.y;
      }
      const double b = ragged_sink(p.sink, h, p.inv_c), root = fabs(b) + sqrt(1.0 + b * b);
      const float a = p.stat[int64_t(h) * p.tokens + block.x + block.z + threadIdx.x] * p.scale;
      double w = (b >= 0.0 ? root : 1.0 / root) * (double(a) / double(p.scale));
      for (int i = 0; i < p.log2n; ++i) w *= w;
      const float ps = float(w);
      l += ps;
      share = l == 0.f ? 0.f : ps * delta / (l * l);
    }
    share = warp_sum(share);
    if (lane == 0) scratch[warp] = share;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const double b = ragged_sink(p.sink, h, p.inv_c);
    const float all = (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
    p.sink_parts[int64_t(p.blocks.prefix[block.w] + (block.z >> 7)) * p.H + h] =
        ctl->abort_flag != 0 ? __int_as_float(0x7fc00000) : float(-double(p.n_f) * double(p.inv_c) / sqrt(1.0 + b * b) * double(all));
    __threadfence();
    const int64_t last = int64_t(n) * p.H - 1;
    scratch[4] = atomicAdd(&p.blocks.header->counter, 1) == last ? 1.f : 0.f;
  }
  __syncthreads();
  if (scratch[4] == 0.f) return;
  __threadfence();
  for (int head = warp; head < p.H; head += int(blockDim.x >> 5)) {
    double sum = 0.0;
    for (int c = lane; c < n; c += 32) sum += double(__ldcg(p.sink_parts + int64_t(c) * p.H + head));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) p.dsink[head] = float(sum);
  }
}

template <int D, int BS, int CTAS>
__global__ void __launch_bounds__(Cfg<D, BS, CTAS>::NTHREADS, CTAS)
ragged_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                   const __grid_constant__ RaggedBwdParams p) {
  using C = Cfg<D, BS, CTAS>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Control* ctl = reinterpret_cast<Control*>(smem + C::CTL_OFF);
  const int warp = threadIdx.x >> 5;
  // The lists are in place when the delta kernel has finished; a CTA behind their end has nothing to set up for.  dK/dV blocks, the
  // dearer kind, come first; the last CTA writes the sinks' gradients where there are no blocks.
  griddep_wait();
  const int n = p.blocks.header->items, kv_ctas = p.blocks.max_items * p.Hkv;
  if (blockIdx.x + 1 == gridDim.x) {
    if (p.dsink != nullptr && n == 0)
      for (int h = threadIdx.x; h < p.H; h += blockDim.x) p.dsink[h] = 0.f;
    return;
  }
  const bool keys = int(blockIdx.x) < kv_ctas;
  const int idx = keys ? int(blockIdx.x) : int(blockIdx.x) - kv_ctas, heads = keys ? p.Hkv : p.H;
  if (idx / heads >= n) return;
  const int4 block = p.blocks.list[(keys ? 0 : n) + idx / heads];

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_q); tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v); tma_prefetch_desc(&tm_do);
    mbar_init(&ctl->res_full, 1); mbar_init(&ctl->never, 1);
    for (int i = 0; i < C::NS; ++i) { mbar_init(&ctl->full[i], 1); mbar_init(&ctl->empty[i], 1); mbar_init(&ctl->vec_full[i], 1); mbar_init(&ctl->clean[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&ctl->s_full[i], 1); mbar_init(&ctl->p_done[i], C::EW_WARPS); }
    mbar_init(&ctl->dp_full, 1);
    mbar_init(&ctl->ds_done, C::EW_WARPS);
    mbar_init(&ctl->acc_full, 1);
    ctl->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (keys) bwd_block<C, D, BS, 1>(smem, ctl, &tm_q, &tm_k, &tm_v, &tm_do, p, block, idx % heads);
  else bwd_block<C, D, BS, 0>(smem, ctl, &tm_q, &tm_k, &tm_v, &tm_do, p, block, idx % heads);

  tc_fence_before();
  __syncthreads();
  if (ctl->abort_flag != 0) {
    spoil_block<D>(p, block, idx % heads, keys);
    if (threadIdx.x == 0) {
      if (p.status != nullptr) atomicExch(p.status, ALG_DEV_TIMEOUT);
      const uint64_t t0 = global_timer_ns();                 // let issued loads land before shared memory is released
      while (global_timer_ns() - t0 < 200000ull) { }
    }
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(ctl->tmem_base, C::TMEM_COLS);
  }
  if (!keys && p.dsink != nullptr) sink_share<C>(smem, ctl, p, block, idx % heads, n);
}

// delta_i = dO_i . (o_i + rest_i), a CTA per head and CHUNK tokens, a row per LPR lanes; zeros to the gradients of rows of no sequence.
constexpr int CHUNK = 64;
template <int D>
__global__ void __launch_bounds__(256) ragged_delta_kernel(const __grid_constant__ RaggedBwdParams p) {
  constexpr int LPR = D / 8, RPW = 32 / LPR, ROWS = CHUNK / 8 / RPW;
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lir = lane % LPR, sub = lane / LPR, h = blockIdx.y;
  const int t0 = blockIdx.x * CHUNK + warp * (CHUNK / 8) + sub;
  int first, last;
  ragged_extent(p.cu, p.S, p.tokens, first, last);
  uint4 g[ROWS], o[ROWS], r[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int64_t t = min(t0 + u * RPW, p.tokens - 1);
    g[u] = __ldg(reinterpret_cast<const uint4*>(p.d_o + t * p.gs.t + h * p.gs.h + lir * 8));
    o[u] = __ldg(reinterpret_cast<const uint4*>(p.o + t * p.os.t + h * p.os.h + lir * 8));
    r[u] = __ldg(reinterpret_cast<const uint4*>(p.rest + (t * p.H + h) * D + lir * 8));
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const __nv_bfloat162 *g2 = reinterpret_cast<const __nv_bfloat162*>(&g[u]), *o2 = reinterpret_cast<const __nv_bfloat162*>(&o[u]),
                         *r2 = reinterpret_cast<const __nv_bfloat162*>(&r[u]);
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = __bfloat1622float2(g2[i]), b = __bfloat1622float2(o2[i]), c = __bfloat1622float2(r2[i]);
      d = fmaf(a.x, b.x + c.x, d);
      d = fmaf(a.y, b.y + c.y, d);
    }
#pragma unroll
    for (int x = LPR / 2; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
    const int t = t0 + u * RPW;
    if (t >= p.tokens) continue;
    if (t < first || t >= last) {
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(p.dq + t * p.dqs.t + h * p.dqs.h + lir * 8) = zero;
      if (h < p.Hkv) {
        *reinterpret_cast<uint4*>(p.dk + t * p.dks.t + h * p.dks.h + lir * 8) = zero;
        *reinterpret_cast<uint4*>(p.dv + t * p.dvs.t + h * p.dvs.h + lir * 8) = zero;
      }
    } else if (lir == 0) {
      p.delta[int64_t(h) * p.tokens + t] = d;
    }
  }
}

int make_map(CUtensorMap* tm, const void* base, const Strides2& s, int H, int tokens, int D, int box_rows) {
  const uint64_t dims[4] = {64, uint64_t(tokens), uint64_t(D / 64), uint64_t(H)};
  const uint64_t strides[3] = {uint64_t(s.t), 64, uint64_t(s.h)};
  const uint32_t box[4] = {64, uint32_t(box_rows), uint32_t(D / 64), 1};
  return make_tmap_bf16(tm, base, 4, dims, strides, box, true);
}

template <int D, int BS, int CTAS>
int launch_d(const RaggedBwdParams& p, cudaStream_t stream) {
  using C = Cfg<D, BS, CTAS>;
  static_assert(CTAS * smem_bytes<C>() <= 232448 - CTAS * 1024, "shared memory budget of an SM");
  static_assert(C::ACC1_COL + D <= C::TMEM_COLS, "tensor-memory budget of a CTA");
  static_assert(BT == BS || C::PANELS == 1, "a resident tile of several boxes has one panel");
  CUtensorMap tq, tk, tv, tdo;
  if (int rc = make_map(&tq, p.q, p.qs, p.H, p.tokens, D, BS)) return rc;
  if (int rc = make_map(&tk, p.k, p.ks, p.Hkv, p.tokens, D, BS)) return rc;
  if (int rc = make_map(&tv, p.v, p.vs, p.Hkv, p.tokens, D, BS)) return rc;
  if (int rc = make_map(&tdo, p.d_o, p.gs, p.H, p.tokens, D, BS)) return rc;
  auto kern = ragged_bwd_kernel<D, BS, CTAS>;
  static PerDeviceOnce configured;
  if (int rc = configured.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem_bytes<C>())); })) return rc;
  const int64_t ctas = int64_t(p.blocks.max_items) * (p.H + p.Hkv) + 1;
  if (ctas > INT32_MAX || p.H > 65535) { set_error("packed attention backward: too many blocks"); return ALG_ERR_UNSUPPORTED; }
  ALG_CUDA_TRY(launch_dependent(ragged_delta_kernel<D>, dim3(unsigned(p.chunks), unsigned(p.H)), dim3(256), 0, stream, p));
  ALG_CUDA_TRY(launch_dependent(kern, dim3(unsigned(ctas)), dim3(C::NTHREADS), smem_bytes<C>(), stream, tq, tk, tv, tdo, p));
  count_launch(2);
  return ALG_OK;
}

constexpr size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace

// delta | sink's partial sums | header | lists | prefix
size_t ragged_bwd_workspace_bytes(int S, int tokens, int H) {
  return align256(size_t(tokens) * H * sizeof(float)) + align256(size_t(ragged_max_blocks(S, tokens)) * H * sizeof(float)) + ragged_blocks_bytes(S, tokens);
}

int launch_ragged_backward(const RaggedBwdParams& params, void* workspace, cudaStream_t stream) {
  RaggedBwdParams p = params;
  unsigned char* at = static_cast<unsigned char*>(workspace);
  p.chunks = (p.tokens + CHUNK - 1) / CHUNK;
  p.delta = reinterpret_cast<float*>(at);
  at += align256(size_t(p.tokens) * p.H * sizeof(float));
  p.sink_parts = reinterpret_cast<float*>(at);
  at += align256(size_t(ragged_max_blocks(p.S, p.tokens)) * p.H * sizeof(float));
  ragged_blocks_carve(&p.blocks, at, p.S, p.tokens);
  p.y_fast = ragged_fast_range(1 << p.log2n) / p.scale;
  if (int rc = launch_ragged_blocks({p.cu, nullptr, p.S, p.tokens, p.tokens}, p.blocks, stream)) return rc;
  return p.D == 64 ? launch_d<64, 64, 2>(p, stream) : launch_d<128, 128, 1>(p, stream);
}

}  // namespace alg
