// Attention over sequences of different lengths: what the plan, the kernels and the C entry points share.
//
// Queries lie packed, (tokens, heads, D), sequence s in rows [cu[s], cu[s + 1]); keys and values lie packed beside them or in the
// pages of a cache.  G = H / Hkv query heads share a key head, and a 128-row query tile holds G heads of 128 / G
// consecutive tokens, row r = token r / G, head r % G, so that a tile's K and V tiles serve the whole group and a chunk of a
// few tokens still fills rows.  Token i of the Lq at the end of a sequence of Lk keys sees keys [0, i + Lk - Lq].
//
// Lengths are device memory, which the host never reads: a plan kernel ahead of the attention turns them into a list of work items,
// longest first, which the persistent CTAs of the attention kernel take from a counter.  What the lengths say is
// clamped to the tensors' extents, so that no value in them leads outside.
#pragma once

#include <math.h>

#include "common.cuh"

namespace alg {

struct RaggedSeqs {
  const int* cu;            // (S + 1), or nullptr: one token a sequence
  const int* kv_lens;       // (S), or nullptr: keys lie packed like the queries, Lk = Lq
  int S, tokens;            // tokens: rows of the packed tensors
  int kv_capacity;          // no sequence has more keys than this
};

// the rows that sequences may have, [first, end): from the first offset to the last
__device__ __forceinline__ void ragged_extent(const int* cu, int S, int tokens, int& first, int& end) {
  first = min(max(__ldg(cu), 0), tokens);
  end = min(max(__ldg(cu + S), first), tokens);
}

// First row and number of the sequence's packed rows, number of its keys.  Offsets that decrease do not lead out of the extent
// either: its rows' keys are those whose norms are taken, and rows outside it are written by the zero tail.
__device__ __forceinline__ void ragged_lengths(const RaggedSeqs& q, int s, int& row0, int& Lq, int& Lk) {
  if (q.cu != nullptr) {
    int first, end;
    ragged_extent(q.cu, q.S, q.tokens, first, end);
    row0 = min(max(__ldg(q.cu + s), first), end);
    Lq = min(max(__ldg(q.cu + s + 1), row0), end) - row0;
  } else {
    row0 = s;
    Lq = 1;
  }
  Lk = q.kv_lens != nullptr ? min(max(__ldg(q.kv_lens + s), 0), q.kv_capacity) : Lq;
}

// 128-key tiles that the tokens up to `end` (exclusive, of this sequence) see: one at least, so that a token that sees nothing
// still has an item that writes its row
__device__ __forceinline__ int ragged_tiles(int Lq, int Lk, int end) {
  const int visible = Lk - Lq + min(end, Lq);
  return visible > 0 ? (visible + 127) >> 7 : 1;
}

struct __align__(16) RaggedItem {
  int row0, Lq, Lk, seq;    // the sequence
  int t0;                   // first token of the block, counted in the sequence
  int k0, nk;               // key tiles [k0, k0 + nk)
  int slot;                 // < 0: the whole item; else this part's slot (times Hkv, plus the head)
};
struct __align__(16) RaggedCombo {   // an item that is cut along the keys, for the kernel that adds its parts up
  int row0, Lq, Lk, t0;
  int slot, parts, pad0, pad1;
};
struct __align__(16) RaggedHeader {
  int items, combos;        // entries of the lists
  int counter;              // next (item, head) to be taken
  int pad;
};

// Workspace of a forward call: header | norms | items | combos | prefix of the sequences' blocks | again | slots.
struct RaggedPlan {
  RaggedHeader* header;
  RaggedItem* items;
  RaggedCombo* combos;
  int* prefix;              // (S + 1)
  int* again;               // (items, heads): after an (item, head) that a CTA weighs again, the one it found before
  float* slots;             // parts' accumulators, (slot, head, 256 rows, D + 4)
  float* norms;             // per CTA of the plan kernel but the first: largest squared row norm of the keys it saw; nullptr: not taken
  int norm_ctas;
  int max_items, max_combos, max_slots;   // slots: of one head
  int block_tokens;         // tokens of an item: two tiles of 128 / G
  int heads;                // Hkv
  int sms;
};

// A list of (sequence, 128-row block), longest first, for the backward kernels: [0, n) by the queries ahead of a key block,
// [n, 2 n) by the keys behind a query block.
struct RaggedBlocks {
  RaggedHeader* header;     // items: entries of each list
  int4* list;               // (row0, L, first row of the block, sequence)
  int* prefix;
  int max_items;
};

struct Strides2 { int64_t t, h; };

// For the self-tests of the waits: how many tiles a CTA loads (all of them as a rule) before its loading warp waits in vain, and how long.
struct WaitLimits {
  unsigned long long budget_ns = 1000000000ull;
  int max_loads = 0x7fffffff;
};

struct RaggedParams {
  RaggedSeqs seqs;
  RaggedPlan plan;
  const void* q;
  const void* k;            // (tokens, Hkv, D) packed, or the pages
  const void* v;
  void* o;
  void* o_lo;               // what the rounding to o left over, dense (tokens, H, D), or nullptr
  float* stat;              // (H, tokens): a with p = (rho(x) a)^n, or nullptr
  const float* sink;
  Strides2 qs, ks, vs, os;
  int64_t k_page, v_page;   // page strides (paged)
  const int* table;         // (S, table_width) page numbers, or nullptr: packed keys
  int64_t table_stride;
  int table_width, page, log2_page, pages;
  int H, Hkv, G, D, log2n;
  int tile_tokens;          // 128 / G
  float scale, inv_c;
  int zero_tail;            // rows of no sequence are written as zeros
  int* status;
  WaitLimits limits;
};

// One token a sequence (paged_token.cu).
struct __align__(16) TokenHead { int s, h, row0, parts; };   // a head that goes on behind the stretch it began in; parts 0: none
struct TokenPlan {
  int groups, heads, grid;  // row groups of a key head; key heads times groups; CTAs
  float* slots;             // two states a CTA: of the head its stretch begins in, of the one it ends in
  TokenHead* heads_open;    // per CTA
  float x_fast;
};
size_t paged_token_workspace_bytes(int S, int Hkv, int G, int D, int64_t keys);
int launch_paged_token(const RaggedParams& p, void* workspace, cudaStream_t stream);

// rho(x) without cancellation, also where x^2 leaves the range
__device__ __forceinline__ float rho_any(float x) {
  const float rad = fmaf(x, x, 1.0f);
  const float T = rad < 3.0e38f ? fmaf(rad, rsqrt_approx(rad), fabsf(x)) : 2.0f * fabsf(x);
  return x >= 0.0f ? T : __fdividef(1.0f, T);
}

// b / c of a sink.  Past 1e30 either way it takes all of the weight or none, as it does there; an infinite one would meet its own
// reference as infinity times zero.  NaN stays.
__device__ __forceinline__ float ragged_sink(const float* sink, int head, float inv_c) {
  const float b = sink[head] * inv_c;
  return b > 1e30f ? 1e30f : b < -1e30f ? -1e30f : b;
}

// |x| up to which weights may go unshifted: rho(x)^n <= 2^64, and the cancellation of x + sqrt(1 + x^2) stays small.  At x < 0 the root, off
// by |x| (2^-22.9 + 2^-25) for the approximate reciprocal root and the rounding of 1 + x^2, leaves rho = 1 / (2 |x|) or more, so that a
// weight loses 2 n x^2 (2^-22.9 + 2^-25) of itself at most: 3.3e-4, at n = 16
inline float ragged_fast_range(int n) {
  const double rho = pow(2.0, 64.0 / n), x = 0.5 * (rho - 1.0 / rho);
  return float(x < 8.0 ? x : 8.0);
}

__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {      // NaN if one of them is
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

struct AppendParams {
  RaggedSeqs seqs;
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  __nv_bfloat16* q_out;
  __nv_bfloat16* k_pages;
  __nv_bfloat16* v_pages;
  const float* q_gain;      // (D) or nullptr
  const float* k_gain;
  const void* cos;          // (>= capacity, D / 2)
  const void* sin;
  Strides2 qs, ks, vs, os, kps, vps;
  int64_t k_page, v_page;
  const int* table;
  int64_t table_stride;
  int page, log2_page, pages;
  int H, Hkv, D;
  int table_dtype;          // of cos and sin: ALG_BF16 or ALG_F32
  float eps;
  int zero_tail;
};
int launch_paged_append(const AppendParams& p, cudaStream_t stream);

struct RaggedBwdParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  const __nv_bfloat16* o;
  const __nv_bfloat16* rest;
  const __nv_bfloat16* d_o;
  const float* stat;        // (H, tokens)
  const float* sink;
  const int* cu;
  __nv_bfloat16* dq;
  __nv_bfloat16* dk;
  __nv_bfloat16* dv;
  float* dsink;
  float* delta;             // (H, tokens)
  float* sink_parts;        // (blocks, H)
  RaggedBlocks blocks;
  Strides2 qs, ks, vs, os, gs, dqs, dks, dvs;
  int S, tokens, H, Hkv, G, D, log2n, chunks;
  float scale, inv_c, n_f, y_fast;
  int* status;
  WaitLimits limits;
};
size_t ragged_bwd_workspace_bytes(int S, int tokens, int H);
int launch_ragged_backward(const RaggedBwdParams& p, void* workspace, cudaStream_t stream);
int ragged_max_blocks(int S, int tokens);
size_t ragged_blocks_bytes(int S, int tokens);
void ragged_blocks_carve(RaggedBlocks* blocks, void* workspace, int S, int tokens);
int launch_ragged_blocks(const RaggedSeqs& seqs, const RaggedBlocks& blocks, cudaStream_t stream);

bool ragged_takes_norms(int tokens, int Hkv);
size_t ragged_plan_bytes(int S, int tokens, int Hkv, int G, int D, bool may_split);
void ragged_plan_carve(RaggedPlan* plan, void* workspace, int S, int tokens, int Hkv, int G, int D, bool may_split, bool norms);
int launch_ragged_plan(const RaggedParams& p, cudaStream_t stream);
int launch_ragged_attention(const RaggedParams& p, cudaStream_t stream);

}  // namespace alg
