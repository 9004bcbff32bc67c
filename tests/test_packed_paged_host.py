"""The packed and paged operators without a GPU: refusals of the C entry points before any launch, argument layouts, workspace
sizes, and the tests' own formulas against automatic differentiation."""

import ctypes as C

import pytest
import torch

import algebraic_transformer_b200 as A
from algebraic_transformer_b200 import _lib as L
import ragged_reference as R


def test_packed_layouts_match_the_structures():
    for fmt, args in ((L.PACKED_ATTN, L.PackedAttnArgs), (L.PACKED_ATTN_BWD, L.PackedAttnBwdArgs), (L.PAGED_ATTN, L.PagedAttnArgs),
                      (L.PAGED_APPEND, L.PagedAppendArgs)):
        assert fmt.size == C.sizeof(args)
    a = L.PagedAttnArgs.from_buffer_copy(L.PAGED_ATTN.pack(*range(1, 9), *range(10, 19), 8.0, 1, 77, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13))
    assert (a.q, a.sink, a.sequences, a.n, a.c, a.zero_tail, a.table_stride) == (1, 8, 10, 18, 8.0, 1, 77)
    assert list(a.k_stride) == [3, 4, 5] and list(a.o_stride) == [9, 10] and (a.workspace, a.workspace_bytes, a.status) == (11, 12, 13)


def refused(fn, a, code, text=""):
    assert fn(a, None) == code and text in L.load().alg_last_error().decode(), L.load().alg_last_error()


def packed(cls=L.PackedAttnArgs, **kw):
    a = cls(q=16, k=16, v=16, o=16, cu_seqlens=16, sequences=1, tokens=8, H=4, Hkv=2, D=64, n=16, c=8.0)
    for name, heads in (("q", 4), ("k", 2), ("v", 2), ("o", 4)):
        setattr(a, name + "_stride", L.I64x2(heads * 64, 64))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_packed_forward_refusals():
    lib = L.load()
    fn = lib.alg_packed_attn_fwd
    refused(fn, L.PackedAttnArgs(), L.ALG_ERR_INVALID, "null")
    refused(fn, packed(D=96), L.ALG_ERR_UNSUPPORTED, "head_dim")
    refused(fn, packed(n=12), L.ALG_ERR_INVALID, "power of two")
    refused(fn, packed(n=64), L.ALG_ERR_INVALID, "power of two")
    refused(fn, packed(c=0.0), L.ALG_ERR_INVALID, "positive")
    refused(fn, packed(c=float("inf")), L.ALG_ERR_INVALID, "finite")
    refused(fn, packed(H=5), L.ALG_ERR_INVALID, "multiple of the key heads")
    refused(fn, packed(H=258), L.ALG_ERR_INVALID, "128 times")
    refused(fn, packed(tokens=-1), L.ALG_ERR_INVALID, "negative")
    refused(fn, packed(sequences=-1), L.ALG_ERR_INVALID, "negative")
    refused(fn, packed(stat=16), L.ALG_ERR_INVALID, "pair")
    refused(fn, packed(q=8), L.ALG_ERR_INVALID, "16-byte")
    for bad in ((0, 64), (-256, 64), (256, 60), (260, 64), (256, 0)):
        refused(fn, packed(q_stride=L.I64x2(*bad)), L.ALG_ERR_INVALID, "16-byte")
    refused(fn, packed(), L.ALG_ERR_WORKSPACE, "workspace")
    # a single row or head may have any stride; then only the workspace is missing
    refused(fn, packed(tokens=1, q_stride=L.I64x2(0, 64)), L.ALG_ERR_WORKSPACE)
    refused(fn, packed(H=1, Hkv=1, k_stride=L.I64x2(64, 1)), L.ALG_ERR_WORKSPACE)


def test_packed_backward_refusals():
    fn = L.load().alg_packed_attn_bwd
    a = packed(L.PackedAttnBwdArgs)
    refused(fn, a, L.ALG_ERR_INVALID, "null")
    for name in ("o_rest", "d_o", "stat", "dq", "dk", "dv"):
        setattr(a, name, 16)
    for name, heads in (("do", 4), ("dq", 4), ("dk", 2), ("dv", 2)):
        setattr(a, name + "_stride", L.I64x2(heads * 64, 64))
    refused(fn, a, L.ALG_ERR_WORKSPACE, "workspace")
    a.sink = 16
    refused(fn, a, L.ALG_ERR_INVALID, "pair")
    a.sink, a.do_stride = None, L.I64x2(0, 0)
    refused(fn, a, L.ALG_ERR_INVALID, "16-byte")


def paged(cls, **kw):
    a = cls(q=16, k_pages=16, v_pages=16, block_table=16, kv_lens=16, cu_seqlens=16, sequences=2, tokens=8, H=4, Hkv=2, D=64, pages=10,
            page_size=32, table_width=4, table_stride=4)
    a.q_stride = L.I64x2(256, 64)
    a.o_stride = L.I64x2(256, 64)
    if cls is L.PagedAttnArgs:
        a.o, a.n, a.c = 16, 16, 8.0
        a.k_stride = a.v_stride = L.I64x3(32 * 128, 128, 64)
    else:
        a.k = a.v = a.q_out = a.cos = a.sin = 16
        a.table_rows, a.table_dtype, a.eps = 128, L.ALG_F32, 1e-5
        a.k_stride = a.v_stride = L.I64x2(128, 64)
        a.kp_stride = a.vp_stride = L.I64x3(32 * 128, 128, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("cls,name", [(L.PagedAttnArgs, "alg_paged_attn_fwd"), (L.PagedAppendArgs, "alg_paged_append")])
def test_paged_refusals(cls, name):
    fn = getattr(L.load(), name)
    refused(fn, cls(), L.ALG_ERR_INVALID, "null")
    refused(fn, paged(cls, D=32), L.ALG_ERR_UNSUPPORTED, "head_dim")
    for page in (8, 24, 48, 100, 65536):
        refused(fn, paged(cls, page_size=page), L.ALG_ERR_UNSUPPORTED, "power of two")
    refused(fn, paged(cls, pages=0), L.ALG_ERR_INVALID, "extents")
    refused(fn, paged(cls, table_width=-1), L.ALG_ERR_INVALID, "extents")
    refused(fn, paged(cls, table_stride=3), L.ALG_ERR_INVALID, "overlap")
    refused(fn, paged(cls, table_width=1 << 27, table_stride=1 << 27), L.ALG_ERR_INVALID, "2^31")
    refused(fn, paged(cls, cu_seqlens=None), L.ALG_ERR_INVALID, "one token")
    refused(fn, paged(cls, v_pages=24), L.ALG_ERR_INVALID, "16-byte")
    if cls is L.PagedAttnArgs:
        refused(fn, paged(cls), L.ALG_ERR_WORKSPACE, "workspace")
        refused(fn, paged(cls, k_stride=L.I64x3(32 * 128, 100, 64)), L.ALG_ERR_INVALID, "16-byte")
    else:
        refused(fn, paged(cls, table_rows=127), L.ALG_ERR_INVALID, "cover")
        refused(fn, paged(cls, eps=0.0), L.ALG_ERR_INVALID, "epsilon")
        refused(fn, paged(cls, table_dtype=7), L.ALG_ERR_INVALID, "tables")
        refused(fn, paged(cls, vp_stride=L.I64x3(0, 128, 64)), L.ALG_ERR_INVALID, "16-byte")


def test_workspace_sizes_do_not_shrink_with_the_problem():
    lib = L.load()
    sizes = [lib.alg_packed_attn_workspace_bytes(packed(tokens=t, sequences=s)) for t, s in ((0, 0), (8, 1), (300, 8), (300, 300))]
    assert sizes == sorted(sizes) and sizes[0] >= 256
    assert lib.alg_packed_attn_workspace_bytes(packed(H=5)) == 0
    one = lib.alg_paged_attn_workspace_bytes(paged(L.PagedAttnArgs, cu_seqlens=None, tokens=2))
    many = lib.alg_paged_attn_workspace_bytes(paged(L.PagedAttnArgs, cu_seqlens=None, tokens=2, table_width=4000))
    assert 0 < one <= many


def test_tensors_on_the_cpu_are_refused():
    q, k = torch.zeros((4, 2, 64), dtype=torch.bfloat16), torch.zeros((4, 1, 64), dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        A.packed_attention(q, k, k, cu)
    pages = torch.zeros((2, 16, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        A.paged_attention(q, pages, pages, torch.zeros((4, 1), dtype=torch.int32), torch.ones(4, dtype=torch.int32))


@pytest.mark.parametrize("with_sink", [True, False])
def test_gradient_formulas_of_the_tests(with_sink):
    """`ragged_reference.packed_gradients` against automatic differentiation of `ragged_reference.packed`, both in 64 bits."""
    g = torch.Generator().manual_seed(3)
    q, k, v, d_o = (torch.randn((9, h, 8), generator=g, dtype=torch.float64) for h in (4, 2, 2, 4))
    sink = torch.randn(4, generator=g, dtype=torch.float64) if with_sink else None
    cu = torch.tensor([1, 5, 5, 9])
    leaves = [t.requires_grad_() for t in (q, k, v)] + ([sink.requires_grad_()] if with_sink else [])

    def loss(q, k, v, sink=None):
        total = 0.0
        for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
            for h in range(4):
                if b > a:
                    o, _ = R.attend(q[a:b, h], k[a:b, h // 2], v[a:b, h // 2], None if sink is None else sink[h], 0, 4, 1.5)
                    total = total + (o * d_o[a:b, h]).sum()
        return total

    want = torch.autograd.grad(loss(*leaves), leaves)
    got, _ = R.packed_gradients(q.detach(), k.detach(), v.detach(), d_o, cu, None if sink is None else sink.detach(), 4, 1.5)
    for a, b in zip(got, want):
        assert float((a - b).abs().max()) < 1e-12
