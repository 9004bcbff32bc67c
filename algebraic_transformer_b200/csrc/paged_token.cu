// One new token of each sequence against its pages: the generation step's attention.
//
// HBM bound: every K and V row is read once for all the G query heads that share it.  The work, all sequences' 64-key units for
// every key head and one more for what a head's end costs, is one long line, sequence by sequence; each CTA takes an equal stretch of it, whatever the lengths, so no
// schedule has to be made: a CTA adds up the lengths (S loads over its threads) and finds where its stretch begins.  A stretch
// covers the end of one (sequence, head), whole ones, and the start of another; states of heads that are not whole go
// to the workspace and a second kernel merges them, launched ahead so that it only has to wait.  (Merged by the CTA that arrives
// last, a head of 19 parts of 8 rows of 128 took 8 us: one SM's reads and code that it meets for the first time.)
//
// Inside a CTA a producer warp streams 32-key K and V tiles, page by page through the block table, into a shared-memory ring that
// runs on over the heads; consumer warps take the tiles in turn, each with a state of its own (maximum m, normaliser l,
// accumulator; weights (rho(x) rho(-m))^n), on mma.sync.m16n8k16:
//   scores   A = the q rows of the group, B = K rows as they lie
//   output   A = the weights straight from the scores' registers, as two bf16 that carry 16 bits of them, B = V through
//            ldmatrix.trans.  Up to 8 rows: both halves in one product, rows 0-7 and 8-15; up to 16: two products.  More
//            query heads to a key head go as several groups of 16, which read the keys again, from L2.
// Measured: four sequences of 22978 to 60001 keys, 16 heads on 2 of 128 (170 MB): 37 us, 4.6 TB/s; 64 sequences of 81 to 4001, 24 heads
// on 8 of 64 (108 MB): 32 us, 3.4 TB/s.  The stream itself goes at 5.3 (head_dim 64) to 6.3 TB/s; some 8 us are launch, line, first tile
// and merge.  A head alone takes 1.7 us in its CTA, the latency of a tile and of the warps' meeting: 1024 sequences of 64 keys, 55 us, are bound
// by that (asking for the next head's q and page numbers ahead of the meeting did not help).
// Unshifted weights go up to 2^64, and with them the sum of finite values may leave the range.  Where a row of a CTA's stretch comes out infinite
// or NaN although its weights are finite, the CTA goes over its stretch once more, max-shifted from the first tile on (weights of 1 at
// most), and writes the rows again that had come out so.
// Rows behind a sequence's end (the rest of its last page) may hold anything: scores there are masked, V is zeroed in registers.
#include "common.cuh"
#include "ragged.cuh"
#include "sm100_ptx.cuh"

#include <math.h>

#include <algorithm>
#include <type_traits>

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
  // 192 KB of K and V tiles per SM; with sixteen rows less, for the sake of the scratch (96 KB in flight still cover 2 us at this
  // SM's share of HBM)
  static constexpr int STAGES = RB == 8 ? 24 / PANELS / CTAS : D == 64 ? 8 : 6;
  static constexpr int CWARPS = D == 64 ? 4 : 6, CONSUMERS = CWARPS * 32, NTHREADS = CONSUMERS + 32;
  static constexpr int ROW = D + 8;                            // floats from row to row of the scratch: no bank conflicts
  static constexpr int SCRATCH = CWARPS * RB * ROW * 4;        // the warps' accumulators
  static_assert(STAGES % CWARPS == 0 && STAGES <= MAX_STAGES && CWARPS <= MAX_CWARPS, "a slot belongs to one warp");
};

template <int RB> struct __align__(16) Control {
  struct { uint64_t full[MAX_STAGES], empty[MAX_STAGES]; } bars[2];             // of the first time over the stretch and of the second
  uint64_t never;
  int abort_flag, overflowed, start_seq, start_len;
  int64_t start_base;                           // units ahead of the first sequence
  int64_t warp_units[MAX_CWARPS + 1];
  float m[MAX_CWARPS][RB], l[MAX_CWARPS][RB];
  float sink[RB];                               // the sinks' weights at the unshifted reference, negative: out of its range
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
// A head's place on the line: its units and one for its end, where the warps' states meet.  (Without, the stretches of short sequences
// were the last to finish: 33.9 against 29.5 us for 64 sequences of 70 to 4001 keys, 24 heads on 8 of 64, no sinks.)
__device__ __forceinline__ int line_of(int len) { return units_of(len) + 1; }

// A CTA's stretch, head by head.
struct Walk {
  int64_t at, end;          // units of the line; a sequence's heads lie one behind the other
  int64_t base;             // units before sequence s
  int s, len, next_len;     // the sequence, its keys, those of the next one (fetched ahead)
  int units;                // of one head of it
  int hh, u0, u1;           // head (and row group), units of the current segment
};
__device__ __forceinline__ int length_of(const RaggedParams& p, int s) {
  return s < p.seqs.S ? min(max(__ldg(p.seqs.kv_lens + s), 0), p.seqs.kv_capacity) : 0;
}
__device__ __forceinline__ bool walk_next(const RaggedParams& p, int heads, Walk& w) {
  for (;;) {
    if (w.at >= w.end) return false;
    if (w.at >= w.base + int64_t(w.units + 1) * heads) {       // every sequence has a place: one step is enough
      w.base += int64_t(w.units + 1) * heads;
      w.len = w.next_len;
      w.units = units_of(w.len);
      ++w.s;
      w.next_len = length_of(p, w.s + 1);
    }
    const int64_t in = w.at - w.base;
    w.hh = int(in / (w.units + 1));
    w.u0 = int(in - int64_t(w.hh) * (w.units + 1));
    if (w.u0 < w.units) break;
    ++w.at;                                                    // a stretch that begins at a head's end
  }
  w.u1 = int(min(int64_t(w.units), w.u0 + (w.end - w.at)));
  w.at += w.u1 - w.u0 + (w.u1 == w.units ? 1 : 0);
  return true;
}

// (rho(x) sigma)^n.  Out of line: it runs where references differ and, per score, in the max-shifted form; the paths that run always
// stay short for it, and code that is met for the first time costs its fetches.
__device__ __noinline__ float rescale(float x, float sigma, int log2n) { return pow2n_rt(rho_any(x) * sigma, log2n); }

// Four columns of a row's state while states with other references join it: a = sum f v, l = sum f l, f = (rho(m_i) rho(-m))^n.
struct State {
  float m, l, ns;           // reference, normaliser, rho(-m)
  float4 a;
  __device__ __forceinline__ void start(const RaggedParams& p, bool with_sink, int head) {
    const bool sunk = with_sink && p.sink != nullptr;
    m = sunk ? ragged_sink(p.sink, head, p.inv_c) : -1e30f;
    l = sunk ? 1.0f : 0.f;                                     // the sink's weight at its own reference
    ns = rho_any(-m);
    a = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void raise(float most, int log2n) {                 // the reference of the states to come
    if (!(most > m)) return;
    ns = rho_any(-most);
    const float f = m > -1e29f ? rescale(m, ns, log2n) : 0.f;
    m = most;
    l *= f; a.x *= f; a.y *= f; a.z *= f; a.w *= f;
  }
  __device__ __forceinline__ float factor(float mi, int log2n) const {
    return mi == m ? 1.0f : mi > -1e29f ? rescale(mi, ns, log2n) : 0.f;
  }
  __device__ __forceinline__ void add(float mi, float li, const float4& v, int log2n) {
    const float f = mi > -1e29f ? factor(mi, log2n) : 0.f;
    if (li != li) l = li;                                      // a wait that ran out, or a NaN score
    if (f == 0.f) return;                                      // nothing was weighed there, or nothing that counts
    l = fmaf(f, li, l);
    a.x = fmaf(f, v.x, a.x); a.y = fmaf(f, v.y, a.y); a.z = fmaf(f, v.z, a.z); a.w = fmaf(f, v.w, a.w);
  }
  __device__ __forceinline__ float4 result() const {
    const float inv = l == 0.f ? 0.f : 1.0f / l;               // a sequence without keys: zero
    return make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
  }
};
__device__ __forceinline__ float largest(const float4& v) { return max3_abs_nan(max3_abs_nan(0.f, v.x, v.y), v.z, v.w); }   // NaN if one is

template <int D, int RB, int LOG2N>
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

  if (threadIdx.x == 0 || threadIdx.x == 32) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&ctl->bars[threadIdx.x >> 5].full[s], 1); mbar_init(&ctl->bars[threadIdx.x >> 5].empty[s], 1); }
    if (threadIdx.x == 0) {
      mbar_init(&ctl->never, 1);
      ctl->abort_flag = ctl->overflowed = 0;
    }
    fence_barrier_init();
  }
  if (threadIdx.x == C::CONSUMERS) { tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v); }
  griddep_wait();
  griddep_launch();                              // the merging kernel's CTAs move in beside these and wait
  // ---- the line: units of all sequences, and the sequence in which this CTA's stretch begins
  const int S = p.seqs.S, per_thread = (S + C::NTHREADS - 1) / C::NTHREADS;
  const int s_first = min(int(threadIdx.x) * per_thread, S), s_last = min(s_first + per_thread, S);
  int64_t mine = 0;
  int len0 = 0;
  for (int s = s_first; s < s_last; ++s) {
    const int len = length_of(p, s);
    if (s == s_first) len0 = len;
    mine += line_of(len);
  }
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
    int s = s_first, len = len0;
    for (;;) {
      const int64_t n = int64_t(line_of(len)) * heads;
      if (begin < base + n) break;
      base += n;
      len = length_of(p, ++s);
    }
    ctl->start_seq = s;
    ctl->start_len = len;
    ctl->start_base = base;
  }
  __syncthreads();
  if (begin >= total) {
    if (threadIdx.x == 0) plan.heads_open[blockIdx.x] = TokenHead{0, 0, 0, 0};
    return;
  }
  const BoundedWait bw{&ctl->abort_flag, 1000000000ull};
  auto run = [&](auto again) {                   // the stretch; again: the second time, in a copy of its own that costs the first nothing
    constexpr bool SECOND = decltype(again)::value;
    auto& bar = ctl->bars[SECOND ? 1 : 0];
    Walk w;
    w.at = begin; w.end = min(begin + per, total);
    w.s = ctl->start_seq; w.len = ctl->start_len; w.base = ctl->start_base;
    w.units = units_of(w.len);
    w.next_len = length_of(p, w.s + 1);
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
          if (tiles >= p.limits.max_loads) { ok = wait_in_vain(&ctl->abort_flag, &ctl->never, p.limits.budget_ns); break; }
          if (!__all_sync(0xffffffffu, bw.wait(&bar.empty[stage], (uint32_t(tiles / STAGES) & 1u) ^ 1u))) { ok = false; break; }
          unsigned char* dst = smem + size_t(stage) * 2 * TILE_BYTES;
          const int live = min(pieces, chunks - c0);
          if (lane == 0) mbar_arrive_expect_tx(&bar.full[stage], uint32_t(live * rows) * (D * 2) * 2);
          __syncwarp();
          // a lane a copy: of K or V, a panel, a piece of a page
          const int piece = lane / (2 * C::PANELS), pn = (lane >> 1) % C::PANELS, v = lane & 1;
          const int page = __shfl_sync(0xffffffffu, number, (c0 + piece - held) & 31);
          if (piece < live) {
            const int row = (k0 + ((c0 + piece) << log2_rows)) & (p.page - 1);
            tma_load_5d(dst + v * TILE_BYTES + pn * PANEL + piece * rows * 128, v ? &tm_v : &tm_k, &bar.full[stage], 0, row, pn, h, page);
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
      const float2 scale2 = make_float2(p.scale, p.scale), one2 = make_float2(1.f, 1.f);
      bool ok = true, first_segment = true;
      TokenHead open = {0, 0, 0, 0};               // the head that begins in this stretch and goes on behind it
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
        float sink = 0.f;                          // of row `lane`, by warp 0: ready when the tiles are
        if (warp == 0 && p.sink != nullptr && lane < live_rows) {
          const float b = ragged_sink(p.sink, h * p.G + row0 + lane, p.inv_c);
          sink = fabsf(b) <= plan.x_fast ? rescale(b, 1.0f, p.log2n) : -1.0f;
        }
        float acc[D / 8][4];                       // RB = 8: rows r of the weights' leading and of their trailing halves
#pragma unroll
        for (int c = 0; c < D / 8; ++c) acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
        // weights are (rho(x) rho(-m_ref))^n: unshifted (m_ref = 0) until a score of the warp's rows leaves the range in which that is safe
        // (|x| <= x_fast keeps them within 2^+-64 and the cancellation of x + sqrt(1 + x^2) below 3.3e-4 of a weight), max-shifted from then on
        float m_ref[NR];
        float2 l_part[NR];
#pragma unroll
        for (int e = 0; e < NR; ++e) { m_ref[e] = 0.f; l_part[e] = make_float2(0.f, 0.f); }
        bool shifted = SECOND, begun = false;
        for (int t = (warp + CWARPS - tiles % CWARPS) % CWARPS; t < n && ok; t += CWARPS) {
          const int number = tiles + t, stage = number % STAGES;
          if (!__all_sync(0xffffffffu, bw.wait(&bar.full[stage], uint32_t(number / STAGES) & 1u))) { ok = false; break; }
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
          const bool tail = live < TILE;
          auto seen = [&](int b, int j) { return 8 * b + 2 * i + j < live; };
          float2 wgt[NR][4];
          float most = 0.f;                        // largest |x| that counts; NaN if there is one
#pragma unroll
          for (int e = 0; e < NR; ++e)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              wgt[e][b] = __fmul2_rn(make_float2(sc[b][2 * e], sc[b][2 * e + 1]), scale2);
              if (tail) {
                if (!seen(b, 0)) wgt[e][b].x = 0.f;
                if (!seen(b, 1)) wgt[e][b].y = 0.f;
              }
              most = max3_abs_nan(most, wgt[e][b].x, wgt[e][b].y);
            }
          if (!SECOND && !shifted) shifted = __any_sync(0xffffffffu, !(most <= plan.x_fast));
          if (!SECOND && !shifted) {
#pragma unroll
            for (int e = 0; e < NR; ++e)
#pragma unroll
              for (int b = 0; b < 4; ++b) {
                const float2 x = wgt[e][b], rad = __ffma2_rn(x, x, one2);
                float2 y = __ffma2_rn(rad, make_float2(rsqrt_approx(rad.x), rsqrt_approx(rad.y)), x);
                if (LOG2N > 0) {
#pragma unroll
                  for (int it = 0; it < LOG2N; ++it) y = __fmul2_rn(y, y);
                } else {
                  for (int it = 0; it < p.log2n; ++it) y = __fmul2_rn(y, y);
                }
                if (tail) {
                  if (!seen(b, 0)) y.x = 0.f;
                  if (!seen(b, 1)) y.y = 0.f;
                }
                wgt[e][b] = y;
                l_part[e] = __fadd2_rn(l_part[e], y);
              }
          } else {
#pragma unroll
            for (int e = 0; e < NR; ++e) {
              float top = -INFINITY;
#pragma unroll
              for (int b = 0; b < 4; ++b) {
                top = seen(b, 0) ? fmaxf(top, wgt[e][b].x) : top;
                top = seen(b, 1) ? fmaxf(top, wgt[e][b].y) : top;
              }
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
              // the first tile's largest score, then the largest so far
              const float m_new = !(top > -INFINITY) ? m_ref[e] : begun ? fmaxf(m_ref[e], top) : top;
              const float ns = rho_any(-m_new), alpha = m_new == m_ref[e] ? 1.0f : rescale(m_ref[e], ns, p.log2n);
              if (begun && __any_sync(0xffffffffu, alpha != 1.0f)) {
                l_part[e].x *= alpha; l_part[e].y *= alpha;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                  acc[c][2 * e] *= alpha; acc[c][2 * e + 1] *= alpha;
                  if (RB == 8) { acc[c][2] *= alpha; acc[c][3] *= alpha; }
                }
              }
              m_ref[e] = m_new;
#pragma unroll
              for (int b = 0; b < 4; ++b) {
                const float2 x = wgt[e][b];
                const float2 y = make_float2(seen(b, 0) ? rescale(x.x, ns, p.log2n) : 0.f,
                                             seen(b, 1) ? rescale(x.y, ns, p.log2n) : 0.f);
                wgt[e][b] = y;
                l_part[e] = __fadd2_rn(l_part[e], y);
              }
            }
          }
          begun = true;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {         // sixteen keys
            uint32_t hi[4], lo[4];                 // A fragments: rows r, r + 8 of keys 2 i, 2 i + 1, then of those 8 further
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int e = 0; e < NR; ++e) {
                const float2 y = wgt[e][2 * ks + g];
                const uint32_t lead = pack_bf16(y.x, y.y), rest = pack_bf16(y.x - __uint_as_float(lead << 16), y.y - __uint_as_float(lead & 0xffff0000u));
                hi[2 * g + e] = lead;
                if (RB == 8) hi[2 * g + 1] = rest;
                else lo[2 * g + e] = rest;
              }
            auto product = [&](auto tailed) {
              const int first = ks * 16 + 2 * i;
              const uint32_t keep0 = (first < live ? 0xffffu : 0u) | (first + 1 < live ? 0xffff0000u : 0u);
              const uint32_t keep1 = (first + 8 < live ? 0xffffu : 0u) | (first + 9 < live ? 0xffff0000u : 0u);
#pragma unroll
              for (int c = 0; c < D / 8; c += 2) { // sixteen columns of V a load
                uint32_t vb[4];
                ldsm4_trans(sv + (c >> 3) * PANEL + ks * 2048 + v_row + (((uint32_t(c & 7) + v_chunk) ^ swz) << 4), vb);
                if (decltype(tailed)::value) { vb[0] &= keep0; vb[1] &= keep1; vb[2] &= keep0; vb[3] &= keep1; }
                mma(acc[c], hi, vb[0], vb[1]);
                mma(acc[c + 1], hi, vb[2], vb[3]);
                if (RB == 16) {
                  mma(acc[c], lo, vb[0], vb[1]);
                  mma(acc[c + 1], lo, vb[2], vb[3]);
                }
              }
            };
            if (tail) product(std::true_type{});
            else product(std::false_type{});
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.empty[stage]);
        }
        tiles += n;
        // ---- the warps' states together: each leaves its own in shared memory, every thread adds up its columns of a row
        if (!first_segment) consumer_sync<C::CONSUMERS>();        // the scratch has been read
        first_segment = false;
#pragma unroll
        for (int e = 0; e < NR; ++e) {
          float l = l_part[e].x + l_part[e].y;
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          if (i == 0) { ctl->m[warp][r + 8 * e] = begun ? m_ref[e] : -1e30f; ctl->l[warp][r + 8 * e] = ok ? l : __int_as_float(0x7fc00000); }
        }
        if (warp == 0 && lane < RB) ctl->sink[lane] = sink;
        if (begun) {
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            float* to = scratch + (warp * RB + r) * C::ROW + c * 8 + 2 * i;
            if (RB == 8) {                         // an infinite V meets a zero trailing half as NaN: the leading half has the answer then
              const float a = isinf(acc[c][0]) ? acc[c][0] : acc[c][0] + acc[c][2], b = isinf(acc[c][1]) ? acc[c][1] : acc[c][1] + acc[c][3];
              *reinterpret_cast<float2*>(to) = make_float2(a, b);
            } else {
              *reinterpret_cast<float2*>(to) = make_float2(acc[c][0], acc[c][1]);
              *reinterpret_cast<float2*>(to + 8 * C::ROW) = make_float2(acc[c][2], acc[c][3]);
            }
          }
        }
        consumer_sync<C::CONSUMERS>();
        const bool whole = w.u0 == 0 && w.u1 == w.units;
        const int kind = w.u0 > 0 ? 0 : 1;
        float* slot = plan.slots + (int64_t(blockIdx.x) * 2 + kind) * (RB * (D + 2));
        for (int x = threadIdx.x; x < live_rows * (D / 4); x += C::CONSUMERS) {
          const int row = x / (D / 4), col = x % (D / 4) * 4;
          State st;
          bool plain = !whole || ctl->sink[row] >= 0.f;          // everything at the unshifted reference, as a rule: sums
#pragma unroll
          for (int wv = 0; wv < CWARPS; ++wv) plain = plain && (ctl->m[wv][row] == 0.f || !(ctl->m[wv][row] > -1e29f));
          if (plain) {
            st.m = 0.f;
            st.l = whole ? ctl->sink[row] : 0.f;
            st.a = make_float4(0.f, 0.f, 0.f, 0.f);
          } else {
            st.start(p, whole, h * p.G + row0 + row);
            float most = ctl->m[0][row];
#pragma unroll
            for (int wv = 1; wv < CWARPS; ++wv) most = fmaxf(most, ctl->m[wv][row]);
            st.raise(most, p.log2n);
          }
#pragma unroll
          for (int wv = 0; wv < CWARPS; ++wv)
            if (ctl->m[wv][row] > -1e29f)
              st.add(ctl->m[wv][row], ctl->l[wv][row], *reinterpret_cast<const float4*>(scratch + (wv * RB + row) * C::ROW + col), p.log2n);
            else if (!ok || ctl->l[wv][row] != 0.f) st.l = __int_as_float(0x7fc00000);       // a wait ran out
          // Out of range as it is written (a bf16 is infinite from half a step above its largest number on), and not for a NaN among its weights?
          // Then the stretch is gone over again, for the rows that hold such numbers.
          const float4 res = whole ? st.result() : st.a;
          __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.o) + w.s * p.os.t + int64_t(h * p.G + row0 + row) * p.os.h + col;
          float4* part = reinterpret_cast<float4*>(slot + row * D + col);
          if (!SECOND) {
            if (st.l == st.l && !(whole ? largest(res) < 0x1.ffp127f : largest(res) <= 0x1.fffffep127f)) ctl->overflowed = 1;
          } else {
            const uint2 old = whole ? *reinterpret_cast<const uint2*>(to) : make_uint2(0u, 0u);
            const float4 held = whole ? make_float4(__uint_as_float(old.x << 16), __uint_as_float(old.x & 0xffff0000u), __uint_as_float(old.y << 16),
                                                    __uint_as_float(old.y & 0xffff0000u))
                                      : *part;
            const unsigned lanes = D == 128 ? 0xffffffffu : 0xffffu << (lane & 16);      // that have this row
            if (!__any_sync(lanes, !(largest(held) <= 0x1.fffffep127f))) continue;
          }
          if (whole) {
            *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(res.x, res.y), pack_bf16(res.z, res.w));
          } else {
            *part = res;
            if (col == 0) *reinterpret_cast<float2*>(slot + RB * D + row * 2) = make_float2(st.m, st.l);
          }
        }
        if (!whole) {
          const int64_t head_end = w.base + int64_t(w.hh) * (w.units + 1) + w.units;
          if (kind == 1) open = TokenHead{w.s, h, row0, int((head_end - 1) / per) - int(blockIdx.x) + 1};
        }
      }
      if (threadIdx.x == 0) plan.heads_open[blockIdx.x] = open;
    }
  };
  run(std::false_type{});
  // by every thread's own word, and before any of them starts again
  const bool overflowed = __syncthreads_or(ctl->overflowed != 0), ended = __syncthreads_or(ctl->abort_flag != 0);
  if (overflowed && !ended) run(std::true_type{});
  __syncthreads();
  if (ctl->abort_flag != 0 && threadIdx.x == 0) {
    if (p.status != nullptr) atomicExch(p.status, ALG_DEV_TIMEOUT);
    const uint64_t t0 = global_timer_ns();       // let issued loads land before the CTA retires
    while (global_timer_ns() - t0 < 200000ull) { }
  }
}

// Merges the parts of a head that goes on behind the stretch it began in: CTA c takes the head that CTA c of the kernel ahead left
// open, a warp a row, a lane D / 32 columns.  References and normalisers come one a lane, 32 parts at a time; accumulators meet at 2^-10 of
// their size, since as many finite ones as there are CTAs may add up to more than fp32 holds.
template <int D, int RB>
__global__ void __launch_bounds__(256) paged_token_merge_kernel(const __grid_constant__ RaggedParams p, const TokenPlan plan) {
  constexpr int CPL = D / 32, SLOT = RB * (D + 2), BATCH = 16;
  griddep_wait();
  const TokenHead head = plan.heads_open[blockIdx.x];
  if (head.parts == 0) return;
  const int lane = threadIdx.x & 31;
  auto slot_of = [&](int part) { return plan.slots + (int64_t(blockIdx.x + part) * 2 + (part > 0 ? 0 : 1)) * SLOT; };
  for (int row = threadIdx.x >> 5; row < min(RB, p.G - head.row0); row += 8) {
    const int h = head.h * p.G + head.row0 + row;
    const float sunk = p.sink != nullptr ? ragged_sink(p.sink, h, p.inv_c) : -1e30f;
    float m = sunk, l = p.sink != nullptr ? 1.0f : 0.f;
    float a[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) a[c] = 0.f;
    for (int p0 = 0; p0 < head.parts; p0 += 32) {
      const int n = min(32, head.parts - p0);
      const float2 ml = lane < n ? __ldcg(reinterpret_cast<const float2*>(slot_of(p0 + lane) + RB * D + row * 2)) : make_float2(-1e30f, 0.f);
      for (int b0 = 0; b0 < n; b0 += BATCH) {
        float v[BATCH][CPL];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const float* src = slot_of(p0 + min(b0 + j, n - 1)) + row * D + lane * CPL;
          if (CPL == 4) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
            v[j][0] = x.x; v[j][1] = x.y; v[j][CPL - 2] = x.z; v[j][CPL - 1] = x.w;
          } else {
            const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
            v[j][0] = x.x; v[j][1] = x.y;
          }
        }
        if (b0 == 0) {                                 // these parts' reference, and what was added up under the old one
          const float top = fmaxf(m, warp_max(ml.x));
          if (top != m) {
            const float f = m > -1e29f ? rescale(m, rho_any(-top), p.log2n) : 0.f;
            l *= f;
#pragma unroll
            for (int c = 0; c < CPL; ++c) a[c] *= f;
            m = top;
          }
        }
        const float f = ml.x == m ? 1.0f : ml.x > -1e29f ? rescale(ml.x, rho_any(-m), p.log2n) : 0.f;
        if (b0 == 0) {
          const bool nan = __any_sync(0xffffffffu, ml.y != ml.y);        // a wait that ran out, or a NaN score
          l += warp_sum(f != 0.f ? f * ml.y : 0.f);
          if (nan) l = __int_as_float(0x7fc00000);
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const float fj = __shfl_sync(0xffffffffu, f, (b0 + j) & 31) * 0x1p-10f;
          if (b0 + j < n && fj != 0.f) {
#pragma unroll
            for (int c = 0; c < CPL; ++c) a[c] = fmaf(fj, v[j][c], a[c]);
          }
        }
      }
    }
    const float inv = sunk != sunk ? sunk : l == 0.f ? 0.f : 1.0f / l;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.o) + head.s * p.os.t + int64_t(h) * p.os.h + lane * CPL;
#pragma unroll
    for (int c = 0; c < CPL; c += 2) *reinterpret_cast<uint32_t*>(out + c) = pack_bf16(a[c] * inv * 0x1p10f, a[c + 1] * inv * 0x1p10f);
  }
}

template <int D, int RB, int LOG2N>
int launch_n(const RaggedParams& p, const TokenPlan& plan, cudaStream_t stream) {
  using C = Cfg<D, RB>;
  static_assert(C::CTAS * (smem_bytes<D, RB>() + 1024) <= 233472, "shared memory of an SM");
  CUtensorMap tm[2];
  for (int i = 0; i < 2; ++i) {
    const Strides2& s = i == 0 ? p.ks : p.vs;
    const uint64_t dims[5] = {64, uint64_t(p.page), uint64_t(D / 64), uint64_t(p.Hkv), uint64_t(p.pages)};
    const uint64_t strides[4] = {uint64_t(s.t), 64, uint64_t(s.h), uint64_t(i == 0 ? p.k_page : p.v_page)};
    const uint32_t box[5] = {64, uint32_t(std::min(p.page, TILE)), 1, 1, 1};
    if (int rc = make_tmap_bf16(&tm[i], i == 0 ? p.k : p.v, 5, dims, strides, box, true, D == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return rc;
  }
  auto kern = paged_token_kernel<D, RB, LOG2N>;
  static PerDeviceOnce configured;
  if (int rc = configured.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem_bytes<D, RB>())); })) return rc;
  ALG_CUDA_TRY(launch_dependent(kern, dim3(plan.grid), dim3(C::NTHREADS), smem_bytes<D, RB>(), stream, tm[0], tm[1], p, plan));
  ALG_CUDA_TRY(launch_dependent(paged_token_merge_kernel<D, RB>, dim3(plan.grid), dim3(256), 0, stream, p, plan));
  count_launch(2);
  return ALG_OK;
}

template <int D, int RB>
int launch(const RaggedParams& p, const TokenPlan& plan, cudaStream_t stream) {
  return p.log2n == 4 ? launch_n<D, RB, 4>(p, plan, stream) : launch_n<D, RB, 0>(p, plan, stream);
}

constexpr size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
// Rows of an mma product: eight, with both halves of the weights in it, or sixteen.
int row_block(int G) { return G <= 8 ? 8 : 16; }
// CTAs: every SM's, but no more than there can be stretches of MIN_UNITS
int token_grid(int S, int Hkv, int G, int D, int64_t keys) {
  const int64_t groups = (G + row_block(G) - 1) / row_block(G), units = std::max<int64_t>(1, (keys + UNIT - 1) / UNIT) + 1;
  const int64_t stretches = (int64_t(S) * Hkv * groups * units + MIN_UNITS - 1) / MIN_UNITS;
  return int(std::max<int64_t>(1, std::min<int64_t>(stretches, int64_t(sm_count()) * (D == 64 ? 2 : 1))));
}

}  // namespace

size_t paged_token_workspace_bytes(int S, int Hkv, int G, int D, int64_t keys) {
  const size_t grid = size_t(token_grid(S, Hkv, G, D, keys));
  return align256(grid * sizeof(TokenHead)) + grid * 2 * row_block(G) * (D + 2) * sizeof(float);
}

int launch_paged_token(const RaggedParams& p, void* workspace, cudaStream_t stream) {
  const int rb = row_block(p.G);
  TokenPlan plan;
  plan.groups = (p.G + rb - 1) / rb;
  plan.heads = p.Hkv * plan.groups;
  plan.grid = token_grid(p.seqs.S, p.Hkv, p.G, p.D, p.seqs.kv_capacity);
  plan.heads_open = static_cast<TokenHead*>(workspace);
  plan.slots = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + align256(plan.grid * sizeof(TokenHead)));
  plan.x_fast = ragged_fast_range(1 << p.log2n);
  if (p.D == 64) return rb == 8 ? launch<64, 8>(p, plan, stream) : launch<64, 16>(p, plan, stream);
  return rb == 8 ? launch<128, 8>(p, plan, stream) : launch<128, 16>(p, plan, stream);
}

}  // namespace alg
