// New tokens into a paged cache: QK RMS-norm and rotation by each token's own position, keys and values to their places.
//
//   q, k:  y = x / sqrt(mean x^2 + eps) * gain, then (y1 c - y2 s, y1 s + y2 c) over the halves, c and s row `position` of the tables
//   v:     as it is
// Token j of the m new ones of a sequence that has kv_len keys with them stands at position kv_len - m + j; its key goes to
// row position % page of page block_table[sequence][position / page].  Everything is formed in fp32 and rounded once.
//
// HBM bound: every row is read once and written once.  A warp takes one token and up to STEPS x 32 / LPR of its rows (q heads, k
// heads, v heads in turn), LPR = D / 8 lanes a row, 16 bytes a lane, all loads issued ahead of the walk from the token to its
// sequence and page, which is the latency to hide: a 32-way search in cu_seqlens (two loads for up to 1024
// sequences), length, table entry.
// Measured: 6043 new tokens of 24 sequences, 16 heads of 128 (152 MB): 37.2 us, 4.1 TB/s; a warp lives for one load, one walk and one store, and
// nothing of the next token is asked for ahead (qk_prep.cu, the same arithmetic without a walk: 5.1 TB/s).  Eight rows a warp instead of four 40.1, two 41.9,
// eight warps a CTA 41.5; held to fewer registers for 8, 10 or 12 CTAs an SM 37.9, 48, 60.7.
#include "common.cuh"
#include "ragged.cuh"

#include <algorithm>

namespace alg {
namespace {

constexpr int STEPS = 4, WARPS = 4;

// the sequence of `token`, or -1; all 32 lanes of a warp
__device__ __forceinline__ int sequence_of_token(const int* cu, int S, int token, int lane) {
  if (S < 1 || token < __ldg(cu) || token >= __ldg(cu + S)) return -1;
  int lo = 0, n = S;                                  // cu[lo] <= token < cu[lo + n]
  while (n > 1) {
    const int step = (n + 31) >> 5, at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, lane * step < n && __ldg(cu + at) <= token);
    const int hit = below ? 31 - __clz(below) : 0;
    lo += hit * step;
    n = min(step, n - hit * step);
  }
  return lo;
}

template <int D, typename Table>
__global__ void __launch_bounds__(WARPS * 32) paged_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int LPR = D / 8, RPW = 32 / LPR, HALF = D / 2;
  griddep_wait();
  const int lane = threadIdx.x & 31, lir = lane % LPR, sub = lane / LPR;
  const int rows = p.H + 2 * p.Hkv, chunks = (rows + STEPS * RPW - 1) / (STEPS * RPW);
  const int64_t unit = int64_t(blockIdx.x) * WARPS + (threadIdx.x >> 5);
  if (unit >= int64_t(p.seqs.tokens) * chunks) return;
  const int token = int(unit / chunks), row0 = int(unit % chunks) * STEPS * RPW;

  uint4 raw[STEPS];
#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    const int r = min(row0 + u * RPW + sub, rows - 1);
    const __nv_bfloat16* src = r < p.H ? p.q + token * p.qs.t + r * p.qs.h
                             : r < p.H + p.Hkv ? p.k + token * p.ks.t + (r - p.H) * p.ks.h : p.v + token * p.vs.t + (r - p.H - p.Hkv) * p.vs.h;
    raw[u] = *reinterpret_cast<const uint4*>(src + lir * 8);
  }

  const int s = p.seqs.cu != nullptr ? sequence_of_token(p.seqs.cu, p.seqs.S, token, lane) : token;
  int position = -1;
  if (s >= 0) {
    int first, Lq, Lk;
    ragged_lengths(p.seqs, s, first, Lq, Lk);
    position = max(__ldg(p.seqs.kv_lens + s), 0) - Lq + token - first;      // by the length as it is given: one past the table is no place
  }
  if (position < 0 || position >= p.seqs.kv_capacity) {                                  // no place in the cache: the row of q is no query either
    if (p.zero_tail) {
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        const int r = row0 + u * RPW + sub;
        if (r < p.H) *reinterpret_cast<uint4*>(p.q_out + token * p.os.t + r * p.os.h + lir * 8) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    return;
  }
  const bool keeps = row0 + STEPS * RPW > p.H;         // some of this warp's rows go to the pages
  const int number = keeps ? __ldg(p.table + s * p.table_stride + (position >> p.log2_page)) : 0;
  const bool inside = unsigned(number) < unsigned(p.pages);
  const int64_t k_at = number * p.k_page + (position & (p.page - 1)) * p.kps.t, v_at = number * p.v_page + (position & (p.page - 1)) * p.vps.t;

  float c[8], sn[8];
  if (row0 < p.H + p.Hkv) {
    const int64_t at = int64_t(position) * HALF + (lir % (LPR / 2)) * 8;
    if constexpr (sizeof(Table) == 4) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 cv = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.cos) + at + i));
        const float4 sv = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.sin) + at + i));
        c[i] = cv.x; c[i + 1] = cv.y; c[i + 2] = cv.z; c[i + 3] = cv.w;
        sn[i] = sv.x; sn[i + 1] = sv.y; sn[i + 2] = sv.z; sn[i + 3] = sv.w;
      }
    } else {
      const uint4 cv = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.cos) + at));
      const uint4 sv = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.sin) + at));
      const __nv_bfloat162 *c2 = reinterpret_cast<const __nv_bfloat162*>(&cv), *s2 = reinterpret_cast<const __nv_bfloat162*>(&sv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = __bfloat1622float2(c2[i]), b = __bfloat1622float2(s2[i]);
        c[2 * i] = a.x; c[2 * i + 1] = a.y; sn[2 * i] = b.x; sn[2 * i + 1] = b.y;
      }
    }
    if (lir < LPR / 2) {                               // the first half subtracts y2 s
#pragma unroll
      for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
    }
  }
#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    const int r = row0 + u * RPW + sub;
    if (row0 + u * RPW >= rows) break;                 // warp-uniform
    uint4 out = raw[u];
    if (row0 + u * RPW < p.H + p.Hkv) {                // warp-uniform: some row of this step is of q or k
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw[u]);
      float x[8], ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(h[i]);
        x[2 * i] = f.x; x[2 * i + 1] = f.y;
        ss = fmaf(f.x, f.x, ss);
        ss = fmaf(f.y, f.y, ss);
      }
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float tau = rsqrtf(ss * (1.0f / D) + p.eps);
      const float* gain = r < p.H ? p.q_gain : p.k_gain;
      if (gain != nullptr) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(gain + lir * 8)), b = __ldg(reinterpret_cast<const float4*>(gain + lir * 8 + 4));
        x[0] *= tau * a.x; x[1] *= tau * a.y; x[2] *= tau * a.z; x[3] *= tau * a.w;
        x[4] *= tau * b.x; x[5] *= tau * b.y; x[6] *= tau * b.z; x[7] *= tau * b.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= tau;
      }
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y0 = __shfl_xor_sync(0xffffffffu, x[2 * i], LPR / 2), y1 = __shfl_xor_sync(0xffffffffu, x[2 * i + 1], LPR / 2);
        w[i] = pack_bf16(fmaf(x[2 * i], c[2 * i], y0 * sn[2 * i]), fmaf(x[2 * i + 1], c[2 * i + 1], y1 * sn[2 * i + 1]));
      }
      if (r < p.H + p.Hkv) out = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (r < p.H) *reinterpret_cast<uint4*>(p.q_out + token * p.os.t + r * p.os.h + lir * 8) = out;
    else if (r < rows && inside) {
      __nv_bfloat16* dst = r < p.H + p.Hkv ? p.k_pages + k_at + (r - p.H) * p.kps.h : p.v_pages + v_at + (r - p.H - p.Hkv) * p.vps.h;
      *reinterpret_cast<uint4*>(dst + lir * 8) = out;
    }
  }
}

template <int D, typename Table>
int launch(const AppendParams& p, cudaStream_t stream) {
  constexpr int RPW = 32 / (D / 8);
  const int64_t chunks = (p.H + 2 * p.Hkv + STEPS * RPW - 1) / (STEPS * RPW), blocks = (int64_t(p.seqs.tokens) * chunks + WARPS - 1) / WARPS;
  if (blocks > INT32_MAX) { set_error("paged append: too many rows"); return ALG_ERR_UNSUPPORTED; }
  ALG_CUDA_TRY(launch_dependent(paged_append_kernel<D, Table>, dim3(unsigned(blocks)), dim3(WARPS * 32), 0, stream, p));
  count_launch();
  return ALG_OK;
}

}  // namespace

int launch_paged_append(const AppendParams& p, cudaStream_t stream) {
  if (p.table_dtype == ALG_F32) return p.D == 64 ? launch<64, float>(p, stream) : launch<128, float>(p, stream);
  return p.D == 64 ? launch<64, __nv_bfloat16>(p, stream) : launch<128, __nv_bfloat16>(p, stream);
}

}  // namespace alg
