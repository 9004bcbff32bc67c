// The plan of a ragged attention call: one CTA reads the lengths and writes the work items, longest first.
//
// An item is two query tiles (2 * 128 / G tokens) of one sequence; heads are not listed, the attention kernel takes every entry
// once per key head.  Entries are placed by a counting sort over 1024 classes of their length in key tiles, so a
// longest-first deal from a counter leaves the CTAs level to about one short item.  Where the longest items would outlast
// an even share of the work (few long sequences), items are cut along the keys into parts whose accumulators a second
// kernel adds up.  Order within a class varies from run to run; results do not depend on it.
#include <algorithm>

#include "common.cuh"
#include "ragged.cuh"

namespace alg {
namespace {

constexpr int NT = 1024, CLASSES = 1024;
// A part is at least this many key tiles long: a part writes its accumulator and the combine kernel reads it back, which
// is the traffic of about four key tiles.
constexpr int MIN_PART = 16, MAX_PARTS = 64;
constexpr int MAX_CUT = 16384;                         // lists longer than this are not cut

__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {   // exclusive; all NT threads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();                                     // warp_sums of the call before are read
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane], s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    warp_sums[lane] = s - w;
    if (lane == 31) warp_sums[32] = s;
  }
  __syncthreads();
  *total = warp_sums[32];
  return warp_sums[warp] + inc - v;
}

// prefix[s] = blocks of the sequences before s; returns their sum.  Saturates far above any list's size.
__device__ int sequence_blocks(const RaggedSeqs& q, int block_tokens, int* prefix, int* warp_sums) {
  int base = 0;
  for (int s0 = 0; s0 < q.S; s0 += NT) {
    const int s = s0 + int(threadIdx.x);
    int n = 0;
    if (s < q.S) {
      int row0, Lq, Lk;
      ragged_lengths(q, s, row0, Lq, Lk);
      n = (Lq + block_tokens - 1) / block_tokens;
    }
    int total;
    const int at = block_scan(n, warp_sums, &total);
    if (s < q.S) prefix[s] = min(base + at, 1 << 29);
    base = min(base + min(total, 1 << 29), 1 << 29);
  }
  if (threadIdx.x == 0) prefix[q.S] = base;
  __syncthreads();
  return base;
}

// the sequence of block i: the last s with prefix[s] <= i that has blocks
__device__ __forceinline__ int sequence_of(const int* prefix, int S, int i) {
  int lo = 0, hi = S;                                  // prefix[lo] <= i < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

// The largest squared norm of the packed keys' rows, by the plan kernel's other CTAs while the first one makes the list.  With that of an
// item's queries (which the attention kernel takes beside its first products) it bounds the item's scores: where the bound is within the
// range of the unshifted weights, no tile's scores have to be looked at, which costs the attention 8 to 12 %.
__device__ __forceinline__ float row_square(const uint4& v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    s = fmaf(f.x, f.x, s);
    s = fmaf(f.y, f.y, s);
  }
  return s;
}
__device__ void take_norms(const RaggedParams& p, float* shared) {
  const RaggedSeqs& q = p.seqs;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lpr = p.D / 8, lir = lane & (lpr - 1), sub = lane / lpr, rpw = 32 / lpr;
  int first, end;
  ragged_extent(q.cu, q.S, q.tokens, first, end);
  const int tokens = end - first;
  const __nv_bfloat16* K = static_cast<const __nv_bfloat16*>(p.k) + first * p.ks.t + lir * 8;
  const unsigned rows = unsigned(tokens) * unsigned(p.Hkv), heads = unsigned(p.Hkv);        // below 2^31: ragged_takes_norms
  float most = 0.f;
  for (unsigned r0 = (unsigned(blockIdx.x - 1) * (NT / 32) + warp) * rpw * 4; r0 < rows; r0 += unsigned(p.plan.norm_ctas) * (NT / 32) * rpw * 4) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned r = min(r0 + u * rpw + sub, rows - 1), token = r / heads;
      v[u] = __ldg(reinterpret_cast<const uint4*>(K + int64_t(token) * p.ks.t + int64_t(r - token * heads) * p.ks.h));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float s = row_square(v[u]);
      for (int o = lpr / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      most = max3_abs_nan(most, s, 0.f);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max3_abs_nan(most, __shfl_xor_sync(0xffffffffu, most, o), 0.f);
  if (lane == 0) shared[warp] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < NT / 32; ++i) most = max3_abs_nan(most, shared[i], 0.f);
    p.plan.norms[blockIdx.x - 1] = most;
  }
}

__global__ void __launch_bounds__(NT) ragged_plan_kernel(const __grid_constant__ RaggedParams params) {
  const RaggedSeqs& q = params.seqs;
  const RaggedPlan& plan = params.plan;
  __shared__ int warp_sums[33], hist[CLASSES], s_max, s_slots, s_combos, s_parts, s_class, s_quota;
  __shared__ unsigned whole[MAX_CUT / 32];
  __shared__ unsigned long long s_cost;
  griddep_wait();                                      // the workspace may be another call's until here
  if (blockIdx.x > 0) {
    take_norms(params, reinterpret_cast<float*>(hist));
    return;
  }
  hist[threadIdx.x] = 0;
  if (threadIdx.x == 0) { s_max = 1; s_cost = 0; s_slots = 0; s_combos = 0; }
  const int n = min(sequence_blocks(q, plan.block_tokens, plan.prefix, warp_sums), plan.max_items);

  struct Block { int row0, Lq, Lk, seq, t0, n1, cost; };
  auto block_at = [&](int i) {
    Block b;
    b.seq = sequence_of(plan.prefix, q.S, i);
    ragged_lengths(q, b.seq, b.row0, b.Lq, b.Lk);
    b.t0 = (i - plan.prefix[b.seq]) * plan.block_tokens;
    b.n1 = ragged_tiles(b.Lq, b.Lk, b.t0 + plan.block_tokens);
    b.cost = b.n1 + (b.Lq - b.t0 > plan.block_tokens / 2 ? ragged_tiles(b.Lq, b.Lk, b.t0 + plan.block_tokens / 2) : 0);
    return b;
  };

  Block mine;                                          // a thread's first block; the others are worked out anew in every pass
  {
    unsigned long long cost = 0;
    int longest = 1;
    for (int i = threadIdx.x; i < n; i += NT) {
      const Block b = block_at(i);
      if (i < NT) mine = b;
      cost += b.cost;
      longest = max(longest, b.n1);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) cost += __shfl_xor_sync(0xffffffffu, cost, o);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if ((threadIdx.x & 31) == 0) { atomicAdd(&s_cost, cost); atomicMax(&s_max, longest); }
  }
  __syncthreads();
  const int longest = s_max;
  auto class_of = [&](int nk) { return CLASSES - 1 - int(int64_t(nk) * (CLASSES - 1) / longest); };

  // Parts.  Where the longest items are more than half of an even share of the work, the CTAs cannot be level: 168 items of 470
  // score tiles over 148 CTAs take as long as 296 would (847 us).  As many of the longest as fill whole rounds stay whole, the
  // others are cut to fill what the share has left over; where the longest is above the share, all are cut, into quarters of a share.
  // Parts are MIN_PART tiles at least, and grow until the slots hold them all.  Which items stay whole is decided by length and,
  // among equals, by their order in the call, never by the order of arrival: a cut item's sums round differently.
  int target = 1 << 30;                                // key tiles of a part
  if (plan.max_slots > 0 && n <= MAX_CUT) {
    const unsigned long long share = s_cost * plan.heads / plan.sms + 1;        // score tiles a CTA would have, two to a key tile
    if ((unsigned long long)longest * 4 > share) {
      const unsigned long long rounds = share / (2ull * longest);
      const int stay = int(min(rounds * plan.sms / plan.heads, (unsigned long long)n));
      target = int(min(rounds > 0 ? max(share - rounds * 2 * longest, share / 16) / 2 : share / 8, 1ull << 28));
      target = max(MIN_PART, target + 1);
      auto length_of = [&](int i) { return i < NT ? mine.n1 : block_at(i).n1; };
      for (int i = threadIdx.x; i < (n + 31) / 32; i += NT) whole[i] = 0u;
      if (stay > 0) {                                  // the `stay` longest: all of the classes ahead of one, the first of that one
        for (int i = threadIdx.x; i < n; i += NT) atomicAdd(&hist[class_of(length_of(i))], 1);
        __syncthreads();
        int total;
        const int at = block_scan(hist[threadIdx.x], warp_sums, &total);
        if (at < stay && at + hist[threadIdx.x] >= stay) { s_class = threadIdx.x; s_quota = stay - at; }
        __syncthreads();
        hist[threadIdx.x] = 0;
        int seen = 0;
        for (int i0 = 0; i0 < n; i0 += NT) {
          const int i = i0 + int(threadIdx.x), c = i < n ? class_of(length_of(i)) : CLASSES;
          int of_class;
          const int rank = seen + block_scan(c == s_class ? 1 : 0, warp_sums, &of_class);
          seen += of_class;
          if (c < s_class || (c == s_class && rank < s_quota)) atomicOr(&whole[i >> 5], 1u << (i & 31));
        }
      }
      for (;;) {
        __syncthreads();
        if (threadIdx.x == 0) s_parts = 0;
        __syncthreads();
        int parts = 0;
        for (int i = threadIdx.x; i < n; i += NT) {
          const int p = (whole[i >> 5] >> (i & 31)) & 1u ? 1 : min((length_of(i) + target - 1) / target, MAX_PARTS);
          if (p > 1) parts += p;
        }
        parts = __reduce_add_sync(0xffffffffu, parts);
        if ((threadIdx.x & 31) == 0 && parts) atomicAdd(&s_parts, parts);
        __syncthreads();
        if (s_parts <= plan.max_slots || target >= (1 << 28)) break;
        target += target / 4 + 1;
      }
    }
  }
  const bool cut = target < (1 << 30);
  auto parts_of = [&](int i, int n1) { return !cut || ((whole[i >> 5] >> (i & 31)) & 1u) ? 1 : min((n1 + target - 1) / target, MAX_PARTS); };
  for (int i = threadIdx.x; i < n; i += NT) {
    const int n1 = i < NT ? mine.n1 : block_at(i).n1, parts = parts_of(i, n1);
    atomicAdd(&hist[class_of((n1 + parts - 1) / parts)], parts);
  }
  __syncthreads();
  int total;
  const int start = block_scan(hist[threadIdx.x], warp_sums, &total);
  __syncthreads();
  hist[threadIdx.x] = start;                           // from now on: the next place of the class
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const Block b = i < NT ? mine : block_at(i);
    const int parts = parts_of(i, b.n1);
    int at = atomicAdd(&hist[class_of((b.n1 + parts - 1) / parts)], parts);
    int slot = -1;
    if (parts > 1) {
      slot = atomicAdd(&s_slots, parts);
      const int c = atomicAdd(&s_combos, 1);
      if (c < plan.max_combos) plan.combos[c] = RaggedCombo{b.row0, b.Lq, b.Lk, b.t0, slot, parts, 0, 0};
    }
    for (int pt = 0; pt < parts; ++pt, ++at) {
      const int k0 = int(int64_t(b.n1) * pt / parts), k1 = int(int64_t(b.n1) * (pt + 1) / parts);
      if (at < plan.max_items) plan.items[at] = RaggedItem{b.row0, b.Lq, b.Lk, b.seq, b.t0, k0, k1 - k0, parts > 1 ? slot + pt : -1};
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) *plan.header = RaggedHeader{min(total, plan.max_items), min(s_combos, plan.max_combos), 0, 0};
}

// The backward's two lists of 128-row blocks: by the rows from the block to the sequence's end (key blocks, seen by these
// queries), by the rows up to the block's end (query blocks, which see these keys).
__global__ void __launch_bounds__(NT) ragged_blocks_kernel(const RaggedSeqs q, const RaggedBlocks blocks) {
  __shared__ int warp_sums[33], hist[2][CLASSES], s_max;
  griddep_wait();
  hist[0][threadIdx.x] = hist[1][threadIdx.x] = 0;
  if (threadIdx.x == 0) s_max = 1;
  const int n = min(sequence_blocks(q, 128, blocks.prefix, warp_sums), blocks.max_items);
  auto block_at = [&](int i) {
    const int s = sequence_of(blocks.prefix, q.S, i);
    int row0, Lq, Lk;
    ragged_lengths(q, s, row0, Lq, Lk);
    return make_int4(row0, Lq, (i - blocks.prefix[s]) * 128, s);
  };
  for (int i = threadIdx.x; i < n; i += NT) atomicMax(&s_max, (block_at(i).y + 127) >> 7);
  __syncthreads();
  const int longest = s_max;
  auto class_of = [&](const int4& b, int list) {
    const int cost = list == 0 ? (b.y - b.z + 127) >> 7 : (b.z >> 7) + 1;
    return CLASSES - 1 - int(int64_t(cost) * (CLASSES - 1) / longest);
  };
  for (int i = threadIdx.x; i < n; i += NT) {
    const int4 b = block_at(i);
    atomicAdd(&hist[0][class_of(b, 0)], 1);
    atomicAdd(&hist[1][class_of(b, 1)], 1);
  }
  __syncthreads();
  for (int list = 0; list < 2; ++list) {
    int total;
    const int start = block_scan(hist[list][threadIdx.x], warp_sums, &total);
    __syncthreads();
    hist[list][threadIdx.x] = start;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const int4 b = block_at(i);
    for (int list = 0; list < 2; ++list) blocks.list[list * n + atomicAdd(&hist[list][class_of(b, list)], 1)] = b;
  }
  if (threadIdx.x == 0) *blocks.header = RaggedHeader{n, 0, 0, 0};
}

constexpr size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct Sizes { int items, slots, combos; };
Sizes plan_sizes(int S, int tokens, int G, int Hkv, bool may_split) {
  const int block = 2 * (128 / G);
  Sizes z{};
  // parts of a quarter of a CTA's share: four or five times the CTAs, over all heads
  z.slots = may_split ? (5 * sm_count() + Hkv - 1) / Hkv : 0;
  z.combos = z.slots / 2;
  z.items = tokens / block + (S < tokens ? S : tokens) + z.slots + 1;
  return z;
}

}  // namespace

// A pass over the keys pays beside the products of more than a tile or two of them.
bool ragged_takes_norms(int tokens, int Hkv) { return tokens > 256 && int64_t(tokens) * Hkv < (int64_t(1) << 30); }

constexpr size_t kNormBytes = 256 * sizeof(float);

size_t ragged_plan_bytes(int S, int tokens, int Hkv, int G, int D, bool may_split) {
  const Sizes z = plan_sizes(S, tokens, G, Hkv, may_split);
  return 256 + kNormBytes + align256(size_t(z.items) * sizeof(RaggedItem)) + align256(size_t(z.combos) * sizeof(RaggedCombo)) +
         align256((size_t(S) + 1) * sizeof(int)) + align256(size_t(z.items) * Hkv * sizeof(int)) +
         size_t(z.slots) * Hkv * 256 * (D + 4) * sizeof(float);
}

void ragged_plan_carve(RaggedPlan* plan, void* workspace, int S, int tokens, int Hkv, int G, int D, bool may_split, bool norms) {
  const Sizes z = plan_sizes(S, tokens, G, Hkv, may_split);
  unsigned char* at = static_cast<unsigned char*>(workspace);
  plan->header = reinterpret_cast<RaggedHeader*>(at);
  at += 256;
  plan->norm_ctas = norms ? std::min(sm_count() - 1, 255) : 0;
  plan->norms = norms ? reinterpret_cast<float*>(at) : nullptr;
  at += kNormBytes;
  plan->items = reinterpret_cast<RaggedItem*>(at);
  at += align256(size_t(z.items) * sizeof(RaggedItem));
  plan->combos = reinterpret_cast<RaggedCombo*>(at);
  at += align256(size_t(z.combos) * sizeof(RaggedCombo));
  plan->prefix = reinterpret_cast<int*>(at);
  at += align256((size_t(S) + 1) * sizeof(int));
  plan->again = reinterpret_cast<int*>(at);
  at += align256(size_t(z.items) * Hkv * sizeof(int));
  plan->slots = reinterpret_cast<float*>(at);
  plan->max_items = z.items; plan->max_combos = z.combos; plan->max_slots = z.slots;
  plan->block_tokens = 2 * (128 / G);
  plan->heads = Hkv;
  plan->sms = sm_count();
}

int launch_ragged_plan(const RaggedParams& p, cudaStream_t stream) {
  ALG_CUDA_TRY(launch_dependent(ragged_plan_kernel, dim3(1 + p.plan.norm_ctas), dim3(NT), 0, stream, p));
  count_launch();
  return ALG_OK;
}

int ragged_max_blocks(int S, int tokens) { return tokens / 128 + (S < tokens ? S : tokens); }

size_t ragged_blocks_bytes(int S, int tokens) {
  return 256 + align256(2 * size_t(ragged_max_blocks(S, tokens)) * sizeof(int4)) + align256((size_t(S) + 1) * sizeof(int));
}

void ragged_blocks_carve(RaggedBlocks* blocks, void* workspace, int S, int tokens) {
  unsigned char* at = static_cast<unsigned char*>(workspace);
  blocks->max_items = ragged_max_blocks(S, tokens);
  blocks->header = reinterpret_cast<RaggedHeader*>(at);
  at += 256;
  blocks->list = reinterpret_cast<int4*>(at);
  at += align256(2 * size_t(blocks->max_items) * sizeof(int4));
  blocks->prefix = reinterpret_cast<int*>(at);
}

int launch_ragged_blocks(const RaggedSeqs& seqs, const RaggedBlocks& blocks, cudaStream_t stream) {
  ALG_CUDA_TRY(launch_dependent(ragged_blocks_kernel, dim3(1), dim3(NT), 0, stream, seqs, blocks));
  count_launch();
  return ALG_OK;
}

}  // namespace alg
