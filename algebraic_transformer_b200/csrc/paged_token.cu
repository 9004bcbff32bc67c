// One new token of each sequence against its pages: the generation step's attention.
//
// HBM bound: every K and V row is read once for all the G query heads that share it.  The work, all sequences' 64-key units for
// every key head, is one long line, sequence by sequence; each CTA takes an equal stretch of it, whatever the lengths, so no
// schedule has to be made: a CTA adds up the lengths (S loads over its threads) and finds where its stretch begins.  A stretch
// covers the end of one (sequence, head), whole ones, and the start of another; states of heads that are not whole go
// to the workspace, and the CTA that arrives last for such a head merges them (arrival words as in decode.cu: they carry the
// call's number, so nothing has to be zeroed).
//
// Inside a CTA a producer warp streams 32-key K and V tiles, page by page through the block table, into a shared-memory ring that
// runs on over the heads; consumer warps take the tiles in turn, each with a state of its own (maximum m, normaliser l,
// accumulator; weights (rho(x) rho(-m))^n), on mma.sync.m16n8k16:
//   scores   A = the q rows of the group, B = K rows as they lie
//   output   A = the weights straight from the scores' registers, as two bf16 that carry 16 bits of them, B = V through
//            ldmatrix.trans.  Up to 8 rows: both halves in one product, rows 0-7 and 8-15; up to 16: two products.  More
//            query heads to a key head go as several groups of 16, which read the keys again, from L2.
// Rows behind a sequence's end (the rest of its last page) may hold anything: scores there are masked, V is zeroed in registers.
#include "common.cuh"
#include "launchers.h"
#include "ragged.cuh"
#include "sm100_ptx.cuh"

#include <algorithm>

namespace alg {
namespace {

using namespace sm100;

constexpr int TILE = 32, UNIT = 64;             // keys of a ring slot; of a unit of work
constexpr int MIN_UNITS = 2;                    // of a stretch: four tiles, one for each warp at least
constexpr int PANEL = TILE * 128;               // 64 columns of a tile, 128-byte swizzle
constexpr int MAX_STAGES = 12, MAX_CWARPS = 6;

// Tile number t lies in slot t % STAGES and belongs to warp t % CWARPS; STAGES is a multiple of CWARPS, so that a slot is one
// warp's, which follows its phases.
template <int D, int RB> struct Cfg {
  static constexpr int CTAS = D == 64 ? 2 : 1;                 // of an SM
  static constexpr int PANELS = D / 64, TILE_BYTES = PANELS * PANEL;
  static constexpr int STAGES = 24 / PANELS / CTAS;            // 192 KB of K and V tiles per SM
  static constexpr int CWARPS = D == 64 ? 4 : 6, CONSUMERS = CWARPS * 32, NTHREADS = CONSUMERS + 32;
  static constexpr int SCRATCH = CWARPS * RB * 32 * 4;         // 32 columns of the warps' accumulators
  static_assert(STAGES % CWARPS == 0 && STAGES <= MAX_STAGES && CWARPS <= MAX_CWARPS, "a slot belongs to one warp");
};

template <int RB> struct __align__(16) Control {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  int abort_flag, tile_ok, last, start_seq;
  int64_t start_base, total;                    // units ahead of the first sequence; of all sequences (one head)
  int64_t warp_units[MAX_CWARPS + 1];
  float m[MAX_CWARPS][RB], l[MAX_CWARPS][RB], f[MAX_CWARPS][RB], row_l[RB], row_m[RB];
};
template <int D, int RB> constexpr size_t smem_bytes() {
  return size_t(Cfg<D, RB>::STAGES) * 2 * Cfg<D, RB>::TILE_BYTES + Cfg<D, RB>::SCRATCH + sizeof(Control<RB>) + 1024;
}

template <int N> __device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ int units_of(int len) { return len > 0 ? (len + UNIT - 1) / UNIT : 1; }

// A CTA's stretch, head by head.
struct Walk {
  int64_t at, end;          // units of the line; a sequence's heads lie one behind the other
  int64_t base;             // units before sequence s
  int s, len, units;        // the sequence, its keys, its units (of one head)
  int hh, u0, u1;           // head (and row group), units of the current segment
};
__device__ __forceinline__ void walk_sequence(const RaggedParams& p, Walk& w) {
  w.len = min(max(__ldg(p.seqs.kv_lens + w.s), 0), p.seqs.kv_capacity);
  w.units = units_of(w.len);
}
__device__ __forceinline__ bool walk_next(const RaggedParams& p, int heads, Walk& w) {
  if (w.at >= w.end) return false;
  while (w.at >= w.base + int64_t(w.units) * heads) {          // every sequence has a unit: at most one step, but for the first
    w.base += int64_t(w.units) * heads;
    ++w.s;
    walk_sequence(p, w);
  }
  const int64_t in = w.at - w.base;
  w.hh = int(in / w.units);
  w.u0 = int(in - int64_t(w.hh) * w.units);
  w.u1 = int(min(int64_t(w.units), w.u0 + (w.end - w.at)));
  w.at += w.u1 - w.u0;
  return true;
}

template <int D, int RB>
__global__ void __launch_bounds__(Cfg<D, RB>::NTHREADS, Cfg<D, RB>::CTAS)
paged_token_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ RaggedParams p,
                   const TokenPlan plan) {
  using C = Cfg<D, RB>;
  constexpr int STAGES = C::STAGES, TILE_BYTES = C::TILE_BYTES, CWARPS = C::CWARPS;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scratch = reinterpret_cast<float*>(smem + size_t(STAGES) * 2 * TILE_BYTES);
  Control<RB>* ctl = reinterpret_cast<Control<RB>*>(smem + size_t(STAGES) * 2 * TILE_BYTES + C::SCRATCH);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = plan.heads;                  // key heads times row groups

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&ctl->full[s], 1); mbar_init(&ctl->empty[s], 1); }
    ctl->abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == C::CONSUMERS) { tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v); }
  griddep_wait();
  // ---- the line: units of all sequences, and the sequence in which this CTA's stretch begins
  const int S = p.seqs.S, per_thread = (S + C::NTHREADS - 1) / C::NTHREADS;
  const int s_first = min(int(threadIdx.x) * per_thread, S), s_last = min(s_first + per_thread, S);
  int64_t mine = 0;
  for (int s = s_first; s < s_last; ++s) mine += units_of(min(max(__ldg(p.seqs.kv_lens + s), 0), p.seqs.kv_capacity));
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) ctl->warp_units[warp] = incl;
  __syncthreads();
  int64_t before = incl - mine, total = 0;
#pragma unroll
  for (int i = 0; i < CWARPS + 1; ++i) {
    if (i < warp) before += ctl->warp_units[i];
    total += ctl->warp_units[i];
  }
  total *= heads;
  const int64_t per = max(int64_t(MIN_UNITS), (total + gridDim.x - 1) / gridDim.x);
  const int64_t begin = per * blockIdx.x;
  if (begin < total && begin >= before * heads && begin < (before + mine) * heads) {
    int64_t base = before * heads;
    int s = s_first;
    for (;; ++s) {
      const int64_t n = int64_t(units_of(min(max(__ldg(p.seqs.kv_lens + s), 0), p.seqs.kv_capacity))) * heads;
      if (begin < base + n) break;
      base += n;
    }
    ctl->start_seq = s;
    ctl->start_base = base;
  }
  __syncthreads();
  if (begin >= total) return;
  const BoundedWait bw{&ctl->abort_flag, 1000000000ull};
  Walk w;
  w.at = begin; w.end = min(begin + per, total);
  w.s = ctl->start_seq; w.base = ctl->start_base;
  walk_sequence(p, w);
  int tiles = 0;                                 // of the heads before the current one

  if (warp == CWARPS) {                          // producer: the whole warp walks, lane 0 issues, lanes hold page numbers
    const int rows = min(p.page, TILE), log2_rows = 31 - __clz(rows), pieces = TILE >> log2_rows;
    bool ok = true;
    while (ok && walk_next(p, heads, w)) {
      const int k0 = w.u0 * UNIT, k1 = min(w.len, w.u1 * UNIT), h = w.hh / plan.groups;
      const int n = k1 > k0 ? (k1 - k0 + TILE - 1) / TILE : 0, chunks = k1 > k0 ? (k1 - k0 + rows - 1) >> log2_rows : 0;
      const int* pages = p.table + w.s * p.table_stride;
      auto number_at = [&](int c) { return c < chunks ? __ldg(pages + ((k0 + (c << log2_rows)) >> p.log2_page)) : 0; };
      int number = number_at(lane), ahead = number_at(32 + lane), held = 0;       // of chunks [held, held + 32) and the next 32
      for (int t = 0; t < n; ++t, ++tiles) {
        const int c0 = t * pieces;
        if (c0 >= held + 32) { held += 32; number = ahead; ahead = number_at(held + 32 + lane); }
        const int stage = tiles % STAGES;
        if (!__all_sync(0xffffffffu, bw.wait(&ctl->empty[stage], (uint32_t(tiles / STAGES) & 1u) ^ 1u))) { ok = false; break; }
        unsigned char* dst = smem + size_t(stage) * 2 * TILE_BYTES;
        const int live = min(pieces, chunks - c0);
        if (lane == 0) mbar_arrive_expect_tx(&ctl->full[stage], uint32_t(live * rows) * (D * 2) * 2);
        for (int i = 0; i < live; ++i) {
          const int page = __shfl_sync(0xffffffffu, number, c0 + i - held);
          if (lane == 0) {
            const int row = (k0 + ((c0 + i) << log2_rows)) & (p.page - 1);
#pragma unroll
            for (int pn = 0; pn < C::PANELS; ++pn) {
              tma_load_5d(dst + pn * PANEL + i * rows * 128, &tm_k, &ctl->full[stage], 0, row, pn, h, page);
              tma_load_5d(dst + TILE_BYTES + pn * PANEL + i * rows * 128, &tm_v, &ctl->full[stage], 0, row, pn, h, page);
            }
          }
        }
        __syncwarp();
      }
    }
  } else {
    const int r = lane >> 2, i = lane & 3;       // row and column pair of an mma result
    const uint32_t ring = smem_u32(smem);
    const uint32_t k_row = uint32_t(lane & 7) * 128, k_chunk = uint32_t(lane >> 3);              // + 8 keys, + 4 chunks
    const uint32_t v_row = uint32_t(((lane >> 3) & 1) * 8 + (lane & 7)) * 128, v_chunk = uint32_t(lane >> 4);   // + 16 keys, + 2
    const uint32_t swz = uint32_t(lane & 7);
    constexpr int NR = RB / 8;                   // rows of this lane: r, and r + 8 where RB = 16
    bool ok = true;
    while (walk_next(p, heads, w)) {
      const int k0 = w.u0 * UNIT, k1 = min(w.len, w.u1 * UNIT), n = k1 > k0 ? (k1 - k0 + TILE - 1) / TILE : 0;
      const int h = w.hh / plan.groups, row0 = (w.hh % plan.groups) * RB, live_rows = min(RB, p.G - row0);
      uint32_t qa[D / 16][4];                    // A fragments of q: rows r, r + 8, columns 2 i, 2 i + 1 and 8 further of each 16
      {
        const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q) + w.s * p.qs.t + int64_t(h * p.G + row0) * p.qs.h;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool there = e < NR && r + 8 * e < live_rows;
          const uint32_t* src = reinterpret_cast<const uint32_t*>(q + int64_t(there ? r + 8 * e : 0) * p.qs.h);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            qa[ks][e] = there ? __ldg(src + ks * 8 + i) : 0u;
            qa[ks][2 + e] = there ? __ldg(src + ks * 8 + 4 + i) : 0u;
          }
        }
      }
      float acc[D / 8][4];                       // RB = 8: rows r of the weights' leading and of their trailing halves
#pragma unroll
      for (int c = 0; c < D / 8; ++c) acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
      float m_ref[NR], shift[NR], l_part[NR];
#pragma unroll
      for (int e = 0; e < NR; ++e) { m_ref[e] = -1e30f; shift[e] = 0.f; l_part[e] = 0.f; }
      for (int t = (warp + CWARPS - tiles % CWARPS) % CWARPS; t < n && ok; t += CWARPS) {
        const int number = tiles + t, stage = number % STAGES;
        if (!__all_sync(0xffffffffu, bw.wait(&ctl->full[stage], uint32_t(number / STAGES) & 1u))) { ok = false; break; }
        const uint32_t sk = ring + uint32_t(stage) * (2 * TILE_BYTES), sv = sk + TILE_BYTES;
        float sc[4][4];
#pragma unroll
        for (int b = 0; b < 4; ++b) sc[b][0] = sc[b][1] = sc[b][2] = sc[b][3] = 0.f;
#pragma unroll
        for (int kq = 0; kq < D / 32; ++kq) {    // 32 columns of K a load
#pragma unroll
          for (int b = 0; b < 4; ++b) {          // eight keys
            uint32_t kb[4];
            ldsm4(sk + (kq >> 1) * PANEL + b * 1024 + k_row + (((uint32_t(kq & 1) * 4 + k_chunk) ^ swz) << 4), kb);
            mma(sc[b], qa[2 * kq], kb[0], kb[1]);
            mma(sc[b], qa[2 * kq + 1], kb[2], kb[3]);
          }
        }
        const int live = k1 - k0 - t * TILE;     // keys of the tile; columns 8 b + 2 i, + 1 are this lane's
        float wgt[NR][8];
#pragma unroll
        for (int e = 0; e < NR; ++e) {
          float top = -1e30f;
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float x = sc[b][2 * e + j] * p.scale;
              wgt[e][2 * b + j] = x;
              top = (8 * b + 2 * i + j < live) ? fmaxf(top, x) : top;
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          if (__any_sync(0xffffffffu, top > m_ref[e])) {
            const float m_new = fmaxf(top, m_ref[e]);
            const float ns = rho_any(-m_new);
            const float alpha = m_new == m_ref[e] ? 1.0f : m_ref[e] > -1e29f ? pow2n_rt(rho_any(m_ref[e]) * ns, p.log2n) : 0.f;
            l_part[e] *= alpha;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
              acc[c][2 * e] *= alpha; acc[c][2 * e + 1] *= alpha;
              if (RB == 8) { acc[c][2] *= alpha; acc[c][3] *= alpha; }
            }
            m_ref[e] = m_new;
            shift[e] = m_new > -1e29f ? ns : 0.f;
          }
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float x = wgt[e][2 * b + j];
              const float y = (8 * b + 2 * i + j < live) ? pow2n_rt(rho_any(x) * shift[e], p.log2n) : 0.f;
              wgt[e][2 * b + j] = y;
              l_part[e] += y;
            }
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {         // sixteen keys
          uint32_t hi[4], lo[4];                 // A fragments: rows r, r + 8 of keys 2 i, 2 i + 1, then of those 8 further
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int e = 0; e < NR; ++e) {
              const float a = wgt[e][4 * ks + 2 * g], b = wgt[e][4 * ks + 2 * g + 1];
              const uint32_t lead = pack_bf16(a, b), rest = pack_bf16(a - __uint_as_float(lead << 16), b - __uint_as_float(lead & 0xffff0000u));
              hi[2 * g + e] = lead;
              if (RB == 8) hi[2 * g + 1] = rest;
              else lo[2 * g + e] = rest;
            }
          const int first = ks * 16 + 2 * i;
          const uint32_t keep0 = (first < live ? 0xffffu : 0u) | (first + 1 < live ? 0xffff0000u : 0u);
          const uint32_t keep1 = (first + 8 < live ? 0xffffu : 0u) | (first + 9 < live ? 0xffff0000u : 0u);
#pragma unroll
          for (int c = 0; c < D / 8; c += 2) {   // sixteen columns of V a load
            uint32_t vb[4];
            ldsm4_trans(sv + (c >> 3) * PANEL + ks * 2048 + v_row + (((uint32_t(c & 7) + v_chunk) ^ swz) << 4), vb);
            if (live < TILE) { vb[0] &= keep0; vb[1] &= keep1; vb[2] &= keep0; vb[3] &= keep1; }
            mma(acc[c], hi, vb[0], vb[1]);
            mma(acc[c + 1], hi, vb[2], vb[3]);
            if (RB == 16) {
              mma(acc[c], lo, vb[0], vb[1]);
              mma(acc[c + 1], lo, vb[2], vb[3]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->empty[stage]);
      }
      tiles += n;
      // ---- the warps' states together
#pragma unroll
      for (int e = 0; e < NR; ++e) {
        l_part[e] += __shfl_xor_sync(0xffffffffu, l_part[e], 1);
        l_part[e] += __shfl_xor_sync(0xffffffffu, l_part[e], 2);
        if (i == 0) { ctl->m[warp][r + 8 * e] = m_ref[e]; ctl->l[warp][r + 8 * e] = ok ? l_part[e] : __int_as_float(0x7fc00000); }
      }
      consumer_sync<C::CONSUMERS>();
      const bool whole = w.u0 == 0 && w.u1 == w.units;
      if (int(threadIdx.x) < RB) {
        const int row = threadIdx.x;
        const bool sunk = whole && p.sink != nullptr && row < live_rows;
        const float bs = sunk ? p.sink[h * p.G + row0 + row] * p.inv_c : -1e30f;
        float mm = bs;
#pragma unroll
        for (int wv = 0; wv < CWARPS; ++wv) mm = fmaxf(mm, ctl->m[wv][row]);
        const float ns = rho_any(-mm);
        float l = sunk ? pow2n_rt(rho_any(bs) * ns, p.log2n) : 0.f;
#pragma unroll
        for (int wv = 0; wv < CWARPS; ++wv) {
          const float mw = ctl->m[wv][row], lw = ctl->l[wv][row];
          const float f = mw == mm ? 1.0f : mw > -1e29f ? pow2n_rt(rho_any(mw) * ns, p.log2n) : 0.f;
          ctl->f[wv][row] = f;
          l += f == 0.f && lw == 0.f ? 0.f : f * lw;
          if (lw != lw) l = lw;                  // a wait that ran out, or a NaN score
        }
        ctl->row_l[row] = l;
        ctl->row_m[row] = mm;
      }
      const int64_t pair = int64_t(w.s) * heads + w.hh;
      float* slot = plan.slots + (int64_t(blockIdx.x) * 2 + (w.u0 > 0 ? 0 : 1)) * (RB * (D + 2));
      for (int c0 = 0; c0 < D; c0 += 32) {
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          if (c * 8 >= c0 && c * 8 < c0 + 32) {
            float* to = scratch + (warp * RB + r) * 32 + c * 8 - c0 + 2 * i;
            if (RB == 8) {                       // an infinite V meets a zero trailing half as NaN: the leading half has the answer then
              const float a = isinf(acc[c][0]) ? acc[c][0] : acc[c][0] + acc[c][2], b = isinf(acc[c][1]) ? acc[c][1] : acc[c][1] + acc[c][3];
              *reinterpret_cast<float2*>(to) = make_float2(a, b);
            } else {
              *reinterpret_cast<float2*>(to) = make_float2(acc[c][0], acc[c][1]);
              *reinterpret_cast<float2*>(to + 8 * 32) = make_float2(acc[c][2], acc[c][3]);
            }
          }
        }
        consumer_sync<C::CONSUMERS>();
        for (int x = threadIdx.x; x < RB * 32; x += C::CONSUMERS) {
          const int row = x >> 5, col = x & 31;
          float a = 0.f;
#pragma unroll
          for (int wv = 0; wv < CWARPS; ++wv) {
            const float f = ctl->f[wv][row];
            if (f != 0.f) a = fmaf(f, scratch[(wv * RB + row) * 32 + col], a);
          }
          if (whole) {
            const float l = ctl->row_l[row];
            if (row < live_rows)
              static_cast<__nv_bfloat16*>(p.o)[w.s * p.os.t + int64_t(h * p.G + row0 + row) * p.os.h + c0 + col] = __float2bfloat16_rn(l == 0.f ? 0.f : a / l);
          } else {
            slot[row * D + c0 + col] = a;
          }
        }
        consumer_sync<C::CONSUMERS>();
      }
      if (whole) continue;
      if (int(threadIdx.x) < RB) {
        slot[RB * D + threadIdx.x * 2] = ctl->row_m[threadIdx.x];
        slot[RB * D + threadIdx.x * 2 + 1] = ctl->row_l[threadIdx.x];
      }
      __threadfence();                           // the state is visible before this CTA counts as arrived
      consumer_sync<C::CONSUMERS>();
      const int64_t pair_begin = w.base + int64_t(w.hh) * w.units;
      const int c_first = int(pair_begin / per), c_last = int((pair_begin + w.units - 1) / per), parts = c_last - c_first + 1;
      if (threadIdx.x == 0) {
        unsigned long long* word = plan.arrivals + pair;
        unsigned long long seen = *reinterpret_cast<volatile unsigned long long*>(word), next;
        for (;;) {                               // at most `parts` contenders
          next = ((seen >> 16) == plan.call) ? seen + 1 : ((plan.call << 16) | 1ull);
          const unsigned long long prev = atomicCAS(word, seen, next);
          if (prev == seen) break;
          seen = prev;
        }
        const bool last = int(next & 0xffffull) == parts;
        ctl->last = last;
        if (last) *reinterpret_cast<volatile unsigned long long*>(word) = 0ull;     // for a replay with the same number
        __threadfence();
      }
      consumer_sync<C::CONSUMERS>();
      if (!ctl->last) continue;
      // ---- the last to arrive merges the parts, in their order
      auto part = [&](int c) { return plan.slots + (int64_t(c_first + c) * 2 + (c > 0 ? 0 : 1)) * (RB * (D + 2)); };
      for (int row = warp; row < live_rows; row += CWARPS) {                         // a warp a row: reference and normaliser
        const bool sunk = p.sink != nullptr;
        const float bs = sunk ? p.sink[h * p.G + row0 + row] * p.inv_c : -1e30f;
        float mm = bs;
        for (int c = lane; c < parts; c += 32) mm = fmaxf(mm, __ldcg(part(c) + RB * D + row * 2));
        mm = warp_max(mm);
        const float ns = rho_any(-mm);
        float l = 0.f;
        bool nan = false;
        for (int c = lane; c < parts; c += 32) {
          const float mc = __ldcg(part(c) + RB * D + row * 2), lc = __ldcg(part(c) + RB * D + row * 2 + 1);
          const float f = mc == mm ? 1.0f : mc > -1e29f ? pow2n_rt(rho_any(mc) * ns, p.log2n) : 0.f;
          nan |= lc != lc;
          if (f != 0.f) l += f * lc;
        }
        l = warp_sum(l) + (sunk ? pow2n_rt(rho_any(bs) * ns, p.log2n) : 0.f);
        if (__any_sync(0xffffffffu, nan)) l = __int_as_float(0x7fc00000);
        float a[D / 32];
#pragma unroll
        for (int e = 0; e < D / 32; ++e) a[e] = 0.f;
        for (int c = 0; c < parts; c += 4) {     // four parts' loads in flight
          float v[4][D / 32], f[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float* src = part(min(c + u, parts - 1));
            const float mc = __ldcg(src + RB * D + row * 2);
            f[u] = c + u >= parts ? 0.f : mc == mm ? 1.0f : mc > -1e29f ? pow2n_rt(rho_any(mc) * ns, p.log2n) : 0.f;
#pragma unroll
            for (int e = 0; e < D / 32; ++e) v[u][e] = __ldcg(src + row * D + e * 32 + lane);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < D / 32; ++e) a[e] = f[u] != 0.f ? fmaf(f[u], v[u][e], a[e]) : a[e];
        }
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.o) + w.s * p.os.t + int64_t(h * p.G + row0 + row) * p.os.h;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) out[e * 32 + lane] = __float2bfloat16_rn(l == 0.f ? 0.f : a[e] / l);
      }
    }
  }
  __syncthreads();
  if (ctl->abort_flag != 0 && threadIdx.x == 0) {
    if (p.status != nullptr) atomicExch(p.status, ALG_DEV_TIMEOUT);
    const uint64_t t0 = global_timer_ns();       // let issued loads land before the CTA retires
    while (global_timer_ns() - t0 < 200000ull) { }
  }
}

template <int D, int RB>
int launch(const RaggedParams& p, const TokenPlan& plan, cudaStream_t stream) {
  using C = Cfg<D, RB>;
  static_assert(C::CTAS * (smem_bytes<D, RB>() + 1024) <= 233472, "shared memory of an SM");
  CUtensorMap tm[2];
  for (int i = 0; i < 2; ++i) {
    const Strides2& s = i == 0 ? p.ks : p.vs;
    const uint64_t dims[5] = {64, uint64_t(p.page), uint64_t(D / 64), uint64_t(p.Hkv), uint64_t(p.pages)};
    const uint64_t strides[4] = {uint64_t(s.t), 64, uint64_t(s.h), uint64_t(i == 0 ? p.k_page : p.v_page)};
    const uint32_t box[5] = {64, uint32_t(std::min(p.page, TILE)), 1, 1, 1};
    if (int rc = make_tmap_bf16(&tm[i], i == 0 ? p.k : p.v, 5, dims, strides, box, true)) return rc;
  }
  auto kern = paged_token_kernel<D, RB>;
  static PerDeviceOnce configured;
  if (int rc = configured.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem_bytes<D, RB>())); })) return rc;
  ALG_CUDA_TRY(launch_dependent(kern, dim3(plan.grid), dim3(C::NTHREADS), smem_bytes<D, RB>(), stream, tm[0], tm[1], p, plan));
  count_launch();
  return ALG_OK;
}

constexpr size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
// Rows of an mma product: eight, with both halves of the weights in it, or sixteen.
int row_block(int G) { return G <= 8 ? 8 : 16; }
// CTAs: every SM's, but no more than there can be stretches of MIN_UNITS
int token_grid(int S, int Hkv, int G, int D, int64_t keys) {
  const int64_t groups = (G + row_block(G) - 1) / row_block(G), units = std::max<int64_t>(1, (keys + UNIT - 1) / UNIT);
  const int64_t stretches = (int64_t(S) * Hkv * groups * units + MIN_UNITS - 1) / MIN_UNITS;
  return int(std::max<int64_t>(1, std::min<int64_t>(stretches, int64_t(sm_count()) * (D == 64 ? 2 : 1))));
}

}  // namespace

size_t paged_token_workspace_bytes(int S, int Hkv, int G, int D, int64_t keys) {
  const int rb = row_block(G), groups = (G + rb - 1) / rb;
  return align256(size_t(token_grid(S, Hkv, G, D, keys)) * 2 * rb * (D + 2) * sizeof(float)) + size_t(S) * Hkv * groups * 8;
}

int launch_paged_token(const RaggedParams& p, void* workspace, cudaStream_t stream) {
  const int rb = row_block(p.G);
  TokenPlan plan;
  plan.groups = (p.G + rb - 1) / rb;
  plan.heads = p.Hkv * plan.groups;
  plan.grid = token_grid(p.seqs.S, p.Hkv, p.G, p.D, p.seqs.kv_capacity);
  plan.slots = static_cast<float*>(workspace);
  plan.arrivals = reinterpret_cast<unsigned long long*>(static_cast<unsigned char*>(workspace) +
                                                        align256(size_t(plan.grid) * 2 * rb * (p.D + 2) * sizeof(float)));
  plan.call = next_call_number();
  if (p.D == 64) return rb == 8 ? launch<64, 8>(p, plan, stream) : launch<64, 16>(p, plan, stream);
  return rb == 8 ? launch<128, 8>(p, plan, stream) : launch<128, 16>(p, plan, stream);
}

}  // namespace alg
