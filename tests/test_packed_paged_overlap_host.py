"""Tensors that the packed and paged operators write and whose rows share elements are refused ahead of any launch; those that are
only read may overlap."""

import pytest

from algebraic_transformer_b200 import _lib as L
from test_packed_paged_host import packed, paged, refused

# (token, head) strides of 8 tokens of 4 heads of 64 whose rows overlap, and some whose rows do not
OVERLAPPING = [(8, 64), (64, 64), (248, 64), (64, 448), (256, 32)]
APART = [(256, 64), (64, 512), (264, 64), (1024, 128), (72, 576)]


def test_packed_output():
    fn = L.load().alg_packed_attn_fwd
    for bad in OVERLAPPING:
        refused(fn, packed(o_stride=L.I64x2(*bad)), L.ALG_ERR_INVALID, "apart")
        refused(fn, packed(q_stride=L.I64x2(*bad)), L.ALG_ERR_WORKSPACE)
    for good in APART:
        refused(fn, packed(o_stride=L.I64x2(*good)), L.ALG_ERR_WORKSPACE)
    refused(fn, packed(tokens=1, o_stride=L.I64x2(8, 64)), L.ALG_ERR_WORKSPACE)       # a single token's stride says nothing
    refused(fn, packed(H=1, Hkv=1, o_stride=L.I64x2(64, 8)), L.ALG_ERR_WORKSPACE)


@pytest.mark.parametrize("name,heads", [("dq", 4), ("dk", 2), ("dv", 2)])
def test_packed_gradients(name, heads):
    fn = L.load().alg_packed_attn_bwd
    a = packed(L.PackedAttnBwdArgs)
    for field in ("o_rest", "d_o", "stat", "dq", "dk", "dv"):
        setattr(a, field, 16)
    for field, h in (("do", 4), ("dq", 4), ("dk", 2), ("dv", 2)):
        setattr(a, field + "_stride", L.I64x2(h * 64, 64))
    refused(fn, a, L.ALG_ERR_WORKSPACE)
    setattr(a, name + "_stride", L.I64x2(heads * 64 - 8, 64))
    refused(fn, a, L.ALG_ERR_INVALID, "apart")
    setattr(a, name + "_stride", L.I64x2(64, 8 * 64))
    refused(fn, a, L.ALG_ERR_WORKSPACE)


def test_paged_output():
    fn = L.load().alg_paged_attn_fwd
    for bad in OVERLAPPING:
        refused(fn, paged(L.PagedAttnArgs, o_stride=L.I64x2(*bad)), L.ALG_ERR_INVALID, "apart")
    for good in APART:
        refused(fn, paged(L.PagedAttnArgs, o_stride=L.I64x2(*good)), L.ALG_ERR_WORKSPACE)
    # pages that are only read may overlap
    refused(fn, paged(L.PagedAttnArgs, k_stride=L.I64x3(128, 128, 64)), L.ALG_ERR_WORKSPACE)


def test_append():
    fn = L.load().alg_paged_append
    for bad in OVERLAPPING:
        refused(fn, paged(L.PagedAppendArgs, o_stride=L.I64x2(*bad)), L.ALG_ERR_INVALID, "apart")
    # 10 pages of 32 rows of 2 heads: page, row and head strides
    for bad in ((128, 128, 64), (32 * 128 - 8, 128, 64), (32 * 128, 64, 64), (32 * 128, 120, 64), (64, 640, 1272)):
        for name in ("kp_stride", "vp_stride"):
            refused(fn, paged(L.PagedAppendArgs, **{name: L.I64x3(*bad)}), L.ALG_ERR_INVALID, "apart")
    none = dict(tokens=0, sequences=0)                     # nothing to launch: a layout that passes the checks is all
    for good in ((32 * 128, 128, 64), (2 * 32 * 128, 128, 64), (64, 640, 32 * 640), (128, 1280, 64), (32 * 128, 64, 32 * 64)):
        for name in ("kp_stride", "vp_stride"):
            assert fn(paged(L.PagedAppendArgs, **none, **{name: L.I64x3(*good)}), None) == L.ALG_OK
