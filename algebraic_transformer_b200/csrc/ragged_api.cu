// C entry points of the attention over packed sequences and paged caches: argument checks, workspace, kernel choice.
#include <limits.h>
#include <math.h>

#include "common.cuh"
#include "launchers.h"
#include "ragged.cuh"

namespace alg {
namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows of `count` vectors must start on 16-byte boundaries, apart from one another where they are written (written_apart); a single one may
// have any stride, which is replaced by one the copies accept.
bool stride_ok(int64_t* s, int64_t count, int64_t dense) {
  if (count <= 1) { *s = dense; return true; }
  return *s > 0 && *s % 8 == 0 && *s < (int64_t(1) << 38);
}
bool strides_ok(Strides2* s, const int64_t given[2], int64_t rows, int64_t heads, int D) {
  *s = {given[0], given[1]};
  return stride_ok(&s->t, rows, int64_t(heads) * D) && stride_ok(&s->h, heads, D);
}

// No two rows of a tensor that is written share an element: each axis steps over all that the axes of smaller strides span.
bool written_apart(int D, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2 = 1, int64_t s2 = 0) {
  int64_t count[3] = {n0, n1, n2}, stride[3] = {s0, s1, s2}, span = D;
  for (int round = 0; round < 3; ++round) {
    int axis = -1;                                     // the smallest stride that is left
    for (int i = 0; i < 3; ++i)
      if (count[i] > 1 && (axis < 0 || stride[i] < stride[axis])) axis = i;
    if (axis < 0) break;
    if (stride[axis] < span) return false;
    span += stride[axis] * (count[axis] - 1);
    count[axis] = 1;
  }
  return true;
}
bool written_apart(const Strides2& s, int64_t rows, int64_t heads, int D) { return written_apart(D, rows, s.t, heads, s.h); }

int check_link(const char* what, int H, int Hkv, int D, int n, float c) {
  if (D != 64 && D != 128) { set_error("%s: head_dim must be 64 or 128, got %d", what, D); return ALG_ERR_UNSUPPORTED; }
  if (n < 2 || n > 32 || ilog2_exact(n) < 0) { set_error("%s: n must be a power of two in [2, 32], got %d", what, n); return ALG_ERR_INVALID; }
  // c^2 D and its reciprocal, times scores within the unshifted range, stay far inside fp32
  if (!(c >= 0x1p-40f && c <= 0x1p40f)) { set_error("%s: scale c must be positive and finite, within 2^-40 and 2^40", what); return ALG_ERR_INVALID; }
  if (H < 1 || Hkv < 1 || H % Hkv != 0 || H / Hkv > 128) {
    set_error("%s: query heads must be a multiple of the key heads, up to 128 times as many (got %d and %d)", what, H, Hkv);
    return ALG_ERR_INVALID;
  }
  return ALG_OK;
}

// Items are cut along the keys only where that can pay: keys for at least two parts, and blocks too few to keep every CTA busy.
bool may_split(int64_t keys, int tokens, int H, int Hkv) {
  const int64_t blocks = tokens / (2 * (128 / (H / Hkv))) + 1;
  return keys > 16 * 128 && blocks * Hkv < int64_t(8) * sm_count();
}

bool limits_ok(const int* status, const WaitLimits& limits) {
  if (status == nullptr || limits.max_loads < 0) { set_error("selftest: status word and a tile count required"); return false; }
  if (limits.budget_ns == 0 || limits.budget_ns > 1000000000ull) { set_error("selftest: budget must be in (0, 1 s]"); return false; }
  return true;
}

}  // namespace
}  // namespace alg

using namespace alg;

extern "C" {

size_t alg_packed_attn_workspace_bytes(const alg_packed_attn_args* a) {
  if (a == nullptr || a->H < 1 || a->Hkv < 1 || a->H % a->Hkv != 0 || a->H / a->Hkv > 128 || a->tokens < 0 || a->sequences < 0) return 0;
  return ragged_plan_bytes(a->sequences, a->tokens, a->Hkv, a->H / a->Hkv, a->D, may_split(a->tokens, a->tokens, a->H, a->Hkv));
}

}  // extern "C"

static int packed_call(const alg_packed_attn_args* a, const WaitLimits& limits, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a == nullptr || a->q == nullptr || a->k == nullptr || a->v == nullptr || a->o == nullptr || a->cu_seqlens == nullptr) {
    set_error("packed attention: null tensor argument");
    return ALG_ERR_INVALID;
  }
  if (int rc = check_link("packed attention", a->H, a->Hkv, a->D, a->n, a->c)) return rc;
  if (a->tokens < 0 || a->sequences < 0) { set_error("packed attention: negative extent"); return ALG_ERR_INVALID; }
  if ((a->stat == nullptr) != (a->o_rest == nullptr)) { set_error("packed attention: stat and o_rest come as a pair"); return ALG_ERR_INVALID; }
  RaggedParams p{};
  if (!strides_ok(&p.qs, a->q_stride, a->tokens, a->H, a->D) || !strides_ok(&p.ks, a->k_stride, a->tokens, a->Hkv, a->D) ||
      !strides_ok(&p.vs, a->v_stride, a->tokens, a->Hkv, a->D) || !strides_ok(&p.os, a->o_stride, a->tokens, a->H, a->D) ||
      !aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o) || !aligned16(a->o_rest) ||
      !written_apart(p.os, a->tokens, a->H, a->D)) {
    set_error("packed attention: rows must start on 16-byte boundaries, those that are written lie apart");
    return ALG_ERR_INVALID;
  }
  const size_t need = alg_packed_attn_workspace_bytes(a);
  if (a->workspace == nullptr || a->workspace_bytes < need || !aligned16(a->workspace)) {
    set_error("packed attention: workspace of %zu bytes (16-byte aligned) required, got %zu", need, a->workspace_bytes);
    return ALG_ERR_WORKSPACE;
  }
  if (a->tokens == 0) return ALG_OK;
  p.G = a->H / a->Hkv;
  ragged_plan_carve(&p.plan, a->workspace, a->sequences, a->tokens, a->Hkv, p.G, a->D, may_split(a->tokens, a->tokens, a->H, a->Hkv),
                    ragged_takes_norms(a->tokens, a->Hkv));
  p.seqs = {a->cu_seqlens, nullptr, a->sequences, a->tokens, a->tokens};
  p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o; p.o_lo = a->o_rest; p.stat = a->stat; p.sink = a->sink;
  p.H = a->H; p.Hkv = a->Hkv; p.D = a->D; p.log2n = ilog2_exact(a->n);
  p.tile_tokens = 128 / p.G;
  p.scale = float(1.0 / (sqrt(double(a->D)) * double(a->c)));
  p.inv_c = 1.0f / a->c;
  p.zero_tail = a->zero_tail != 0;
  p.status = a->status;
  p.limits = limits;
  return launch_ragged_attention(p, stream);
}

extern "C" {

int alg_packed_attn_fwd(const alg_packed_attn_args* a, void* stream) { return packed_call(a, WaitLimits{}, stream); }

int alg_selftest_packed_timeout(const alg_packed_attn_args* a, int max_loads, unsigned long long budget_ns, void* stream) {
  const WaitLimits limits{budget_ns, max_loads};
  return a != nullptr && !limits_ok(a->status, limits) ? ALG_ERR_INVALID : packed_call(a, limits, stream);
}

size_t alg_packed_attn_bwd_workspace_bytes(const alg_packed_attn_bwd_args* a) {
  if (a == nullptr || a->tokens < 0 || a->sequences < 0 || a->H < 1) return 0;
  return ragged_bwd_workspace_bytes(a->sequences, a->tokens, a->H);
}

}  // extern "C"

static int packed_bwd_call(const alg_packed_attn_bwd_args* a, const WaitLimits& limits, void* stream) {
  if (a == nullptr || a->q == nullptr || a->k == nullptr || a->v == nullptr || a->o == nullptr || a->o_rest == nullptr || a->d_o == nullptr ||
      a->stat == nullptr || a->cu_seqlens == nullptr || a->dq == nullptr || a->dk == nullptr || a->dv == nullptr) {
    set_error("packed attention backward: null tensor argument");
    return ALG_ERR_INVALID;
  }
  if (int rc = check_link("packed attention backward", a->H, a->Hkv, a->D, a->n, a->c)) return rc;
  if (a->tokens < 0 || a->sequences < 0) { set_error("packed attention backward: negative extent"); return ALG_ERR_INVALID; }
  if ((a->sink == nullptr) != (a->dsink == nullptr)) { set_error("packed attention backward: sink and dsink come as a pair"); return ALG_ERR_INVALID; }
  RaggedBwdParams p{};
  if (!strides_ok(&p.qs, a->q_stride, a->tokens, a->H, a->D) || !strides_ok(&p.ks, a->k_stride, a->tokens, a->Hkv, a->D) ||
      !strides_ok(&p.vs, a->v_stride, a->tokens, a->Hkv, a->D) || !strides_ok(&p.os, a->o_stride, a->tokens, a->H, a->D) ||
      !strides_ok(&p.gs, a->do_stride, a->tokens, a->H, a->D) || !strides_ok(&p.dqs, a->dq_stride, a->tokens, a->H, a->D) ||
      !strides_ok(&p.dks, a->dk_stride, a->tokens, a->Hkv, a->D) || !strides_ok(&p.dvs, a->dv_stride, a->tokens, a->Hkv, a->D) ||
      !aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o) || !aligned16(a->o_rest) || !aligned16(a->d_o) ||
      !aligned16(a->dq) || !aligned16(a->dk) || !aligned16(a->dv) || !written_apart(p.dqs, a->tokens, a->H, a->D) ||
      !written_apart(p.dks, a->tokens, a->Hkv, a->D) || !written_apart(p.dvs, a->tokens, a->Hkv, a->D)) {
    set_error("packed attention backward: rows must start on 16-byte boundaries, those that are written lie apart");
    return ALG_ERR_INVALID;
  }
  const size_t need = alg_packed_attn_bwd_workspace_bytes(a);
  if (a->workspace == nullptr || a->workspace_bytes < need || !aligned16(a->workspace)) {
    set_error("packed attention backward: workspace of %zu bytes (16-byte aligned) required, got %zu", need, a->workspace_bytes);
    return ALG_ERR_WORKSPACE;
  }
  if (a->tokens == 0) {
    if (a->dsink != nullptr) ALG_CUDA_TRY(cudaMemsetAsync(a->dsink, 0, size_t(a->H) * sizeof(float), static_cast<cudaStream_t>(stream)));
    return ALG_OK;
  }
  p.q = static_cast<const __nv_bfloat16*>(a->q); p.k = static_cast<const __nv_bfloat16*>(a->k); p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.o = static_cast<const __nv_bfloat16*>(a->o); p.rest = static_cast<const __nv_bfloat16*>(a->o_rest);
  p.d_o = static_cast<const __nv_bfloat16*>(a->d_o);
  p.stat = a->stat; p.sink = a->sink; p.cu = a->cu_seqlens;
  p.dq = static_cast<__nv_bfloat16*>(a->dq); p.dk = static_cast<__nv_bfloat16*>(a->dk); p.dv = static_cast<__nv_bfloat16*>(a->dv);
  p.dsink = a->dsink;
  p.S = a->sequences; p.tokens = a->tokens; p.H = a->H; p.Hkv = a->Hkv; p.G = a->H / a->Hkv; p.D = a->D;
  p.log2n = ilog2_exact(a->n);
  p.scale = float(1.0 / (sqrt(double(a->D)) * double(a->c)));
  p.inv_c = 1.0f / a->c;
  p.n_f = float(a->n);
  p.status = a->status;
  p.limits = limits;
  return launch_ragged_backward(p, a->workspace, static_cast<cudaStream_t>(stream));
}

extern "C" {

int alg_packed_attn_bwd(const alg_packed_attn_bwd_args* a, void* stream) { return packed_bwd_call(a, WaitLimits{}, stream); }

int alg_selftest_packed_bwd_timeout(const alg_packed_attn_bwd_args* a, int max_loads, unsigned long long budget_ns, void* stream) {
  const WaitLimits limits{budget_ns, max_loads};
  return a != nullptr && !limits_ok(a->status, limits) ? ALG_ERR_INVALID : packed_bwd_call(a, limits, stream);
}

}  // extern "C"

template <class Args> static int paged_checks(const Args* a, const char* what) {
  if (a->tokens < 0 || a->sequences < 0 || a->pages < 1 || a->table_width < 0) { set_error("%s: bad extents", what); return ALG_ERR_INVALID; }
  if (a->page_size < 16 || a->page_size > 32768 || ilog2_exact(a->page_size) < 0) {
    set_error("%s: pages of a power of two of tokens, at least 16, got %d", what, a->page_size);
    return ALG_ERR_UNSUPPORTED;
  }
  if (int64_t(a->table_width) * a->page_size > INT_MAX - 4096) { set_error("%s: a sequence's pages hold more keys than 2^31", what); return ALG_ERR_INVALID; }
  if (a->table_width > 0 && a->sequences > 1 && a->table_stride < a->table_width) { set_error("%s: rows of the block table overlap", what); return ALG_ERR_INVALID; }
  if (a->cu_seqlens == nullptr && a->tokens != a->sequences) { set_error("%s: without cu_seqlens every sequence has one token", what); return ALG_ERR_INVALID; }
  return ALG_OK;
}

extern "C" {

size_t alg_paged_attn_workspace_bytes(const alg_paged_attn_args* a) {
  if (a == nullptr || a->H < 1 || a->Hkv < 1 || a->H % a->Hkv != 0 || a->H / a->Hkv > 128 || a->tokens < 0 || a->sequences < 0) return 0;
  if (a->cu_seqlens == nullptr)
    return paged_token_workspace_bytes(a->sequences, a->Hkv, a->H / a->Hkv, a->D, int64_t(a->table_width) * a->page_size);
  return ragged_plan_bytes(a->sequences, a->tokens, a->Hkv, a->H / a->Hkv, a->D,
                           may_split(int64_t(a->table_width) * a->page_size, a->tokens, a->H, a->Hkv));
}

}  // extern "C"

static int paged_call(const alg_paged_attn_args* a, const WaitLimits& limits, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a == nullptr || a->q == nullptr || a->k_pages == nullptr || a->v_pages == nullptr || a->o == nullptr || a->kv_lens == nullptr ||
      a->block_table == nullptr) {
    set_error("paged attention: null tensor argument");
    return ALG_ERR_INVALID;
  }
  if (int rc = check_link("paged attention", a->H, a->Hkv, a->D, a->n, a->c)) return rc;
  if (int rc = paged_checks(a, "paged attention")) return rc;
  RaggedParams p{};
  int64_t kp = a->k_stride[0], vp = a->v_stride[0];
  const int64_t page_elems = int64_t(a->page_size) * a->Hkv * a->D;
  if (!strides_ok(&p.qs, a->q_stride, a->tokens, a->H, a->D) || !strides_ok(&p.ks, a->k_stride + 1, a->page_size, a->Hkv, a->D) ||
      !strides_ok(&p.vs, a->v_stride + 1, a->page_size, a->Hkv, a->D) || !strides_ok(&p.os, a->o_stride, a->tokens, a->H, a->D) ||
      !stride_ok(&kp, a->pages, page_elems) || !stride_ok(&vp, a->pages, page_elems) || !aligned16(a->q) || !aligned16(a->k_pages) ||
      !aligned16(a->v_pages) || !aligned16(a->o) || !written_apart(p.os, a->tokens, a->H, a->D)) {
    set_error("paged attention: rows must start on 16-byte boundaries, those that are written lie apart");
    return ALG_ERR_INVALID;
  }
  const size_t need = alg_paged_attn_workspace_bytes(a);
  if (a->workspace == nullptr || a->workspace_bytes < need || !aligned16(a->workspace)) {
    set_error("paged attention: workspace of %zu bytes (16-byte aligned) required, got %zu", need, a->workspace_bytes);
    return ALG_ERR_WORKSPACE;
  }
  if (a->tokens == 0) return ALG_OK;
  const int64_t keys = int64_t(a->table_width) * a->page_size;
  p.G = a->H / a->Hkv;
  p.seqs = {a->cu_seqlens, a->kv_lens, a->sequences, a->tokens, int(keys)};
  p.q = a->q; p.k = a->k_pages; p.v = a->v_pages; p.o = a->o; p.sink = a->sink;
  p.k_page = kp; p.v_page = vp;
  p.table = a->block_table; p.table_stride = a->table_stride; p.table_width = a->table_width;
  p.page = a->page_size; p.log2_page = ilog2_exact(a->page_size); p.pages = a->pages;
  p.H = a->H; p.Hkv = a->Hkv; p.D = a->D; p.log2n = ilog2_exact(a->n);
  p.tile_tokens = 128 / p.G;
  p.scale = float(1.0 / (sqrt(double(a->D)) * double(a->c)));
  p.inv_c = 1.0f / a->c;
  p.status = a->status;
  p.limits = limits;
  if (a->cu_seqlens == nullptr) return launch_paged_token(p, a->workspace, stream);
  ragged_plan_carve(&p.plan, a->workspace, a->sequences, a->tokens, a->Hkv, p.G, a->D, may_split(keys, a->tokens, a->H, a->Hkv), false);
  p.zero_tail = a->zero_tail != 0;
  return launch_ragged_attention(p, stream);
}

extern "C" {

int alg_paged_attn_fwd(const alg_paged_attn_args* a, void* stream) { return paged_call(a, WaitLimits{}, stream); }

int alg_selftest_paged_timeout(const alg_paged_attn_args* a, int max_loads, unsigned long long budget_ns, void* stream) {
  const WaitLimits limits{budget_ns, max_loads};
  return a != nullptr && !limits_ok(a->status, limits) ? ALG_ERR_INVALID : paged_call(a, limits, stream);
}

int alg_paged_append(const alg_paged_append_args* a, void* stream_) {
  if (a == nullptr || a->q == nullptr || a->k == nullptr || a->v == nullptr || a->q_out == nullptr || a->k_pages == nullptr ||
      a->v_pages == nullptr || a->kv_lens == nullptr || a->block_table == nullptr || a->cos == nullptr || a->sin == nullptr) {
    set_error("paged append: null tensor argument");
    return ALG_ERR_INVALID;
  }
  if (a->D != 64 && a->D != 128) { set_error("paged append: head_dim must be 64 or 128, got %d", a->D); return ALG_ERR_UNSUPPORTED; }
  if (a->H < 1 || a->Hkv < 1 || a->H > (1 << 20) || a->Hkv > (1 << 20)) { set_error("paged append: bad extents"); return ALG_ERR_INVALID; }
  if (int rc = paged_checks(a, "paged append")) return rc;
  if (!(a->eps > 0.0f)) { set_error("paged append: epsilon must be positive"); return ALG_ERR_INVALID; }
  if (a->table_dtype != ALG_BF16 && a->table_dtype != ALG_F32) { set_error("paged append: rotation tables are bf16 or fp32"); return ALG_ERR_INVALID; }
  const int64_t keys = int64_t(a->table_width) * a->page_size;
  if (a->table_rows < keys) {
    set_error("paged append: the rotation tables must cover the %lld positions of a sequence's pages, got %d rows", (long long)keys, a->table_rows);
    return ALG_ERR_INVALID;
  }
  AppendParams p{};
  p.k_page = a->kp_stride[0]; p.v_page = a->vp_stride[0];
  const int64_t page_elems = int64_t(a->page_size) * a->Hkv * a->D;
  if (!strides_ok(&p.qs, a->q_stride, a->tokens, a->H, a->D) || !strides_ok(&p.ks, a->k_stride, a->tokens, a->Hkv, a->D) ||
      !strides_ok(&p.vs, a->v_stride, a->tokens, a->Hkv, a->D) || !strides_ok(&p.os, a->o_stride, a->tokens, a->H, a->D) ||
      !strides_ok(&p.kps, a->kp_stride + 1, a->page_size, a->Hkv, a->D) || !strides_ok(&p.vps, a->vp_stride + 1, a->page_size, a->Hkv, a->D) ||
      !stride_ok(&p.k_page, a->pages, page_elems) || !stride_ok(&p.v_page, a->pages, page_elems) || !aligned16(a->q) || !aligned16(a->k) ||
      !aligned16(a->v) || !aligned16(a->q_out) || !aligned16(a->k_pages) || !aligned16(a->v_pages) || !aligned16(a->cos) || !aligned16(a->sin) ||
      !aligned16(a->q_gain) || !aligned16(a->k_gain) || !written_apart(p.os, a->tokens, a->H, a->D) ||
      !written_apart(a->D, a->pages, p.k_page, a->page_size, p.kps.t, a->Hkv, p.kps.h) ||
      !written_apart(a->D, a->pages, p.v_page, a->page_size, p.vps.t, a->Hkv, p.vps.h)) {
    set_error("paged append: rows, gains and tables must start on 16-byte boundaries, rows that are written lie apart");
    return ALG_ERR_INVALID;
  }
  if (a->tokens == 0) return ALG_OK;
  p.seqs = {a->cu_seqlens, a->kv_lens, a->sequences, a->tokens, int(keys)};
  p.q = static_cast<const __nv_bfloat16*>(a->q); p.k = static_cast<const __nv_bfloat16*>(a->k); p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
  p.k_pages = static_cast<__nv_bfloat16*>(a->k_pages); p.v_pages = static_cast<__nv_bfloat16*>(a->v_pages);
  p.q_gain = a->q_gain; p.k_gain = a->k_gain; p.cos = a->cos; p.sin = a->sin;
  p.table = a->block_table; p.table_stride = a->table_stride;
  p.page = a->page_size; p.log2_page = ilog2_exact(a->page_size); p.pages = a->pages;
  p.H = a->H; p.Hkv = a->Hkv; p.D = a->D; p.table_dtype = a->table_dtype; p.eps = a->eps;
  p.zero_tail = a->zero_tail != 0;
  return launch_paged_append(p, static_cast<cudaStream_t>(stream_));
}

}  // extern "C"
