"""Packed attention where a CTA takes many items of one key tile, one after the other: every hand-over of a query tile and of its row
norm is then an item's first and last."""

import pytest
import torch

import algebraic_transformer_b200 as A
from algebraic_transformer_b200 import _lib as L
import ragged_reference as R
from test_gpu_packed_attention import make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def with_status(q, k, v, sink, cu):
    """The call through the C ABI, which has a status word."""
    lib, (T, H, D), Hkv = L.load(), q.shape, k.shape[1]
    o, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device=DEV)
    a = L.PackedAttnArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=o.data_ptr(), cu_seqlens=cu.data_ptr(), sink=sink.data_ptr(),
                         sequences=cu.numel() - 1, tokens=T, H=H, Hkv=Hkv, D=D, n=16, c=8.0, zero_tail=1, status=status.data_ptr())
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o)):
        setattr(a, name + "_stride", L.I64x2(*t.stride()[:2]))
    ws = torch.empty(lib.alg_packed_attn_workspace_bytes(a), dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    assert lib.alg_packed_attn_fwd(a, torch.cuda.current_stream().cuda_stream) == L.ALG_OK
    torch.cuda.synchronize()
    return o, int(status)


@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 64), (6, 2, 64), (8, 2, 128)])
def test_many_items_of_one_key_tile(H, Hkv, D):
    lens = [1 + (37 * i) % 128 for i in range(900)]
    q, k, v, sink, cu = make(lens, H, Hkv, D, seed=D + H)
    ref, spread, err = R.packed(q, k, v, cu, sink, 16, 8.0)
    first = None
    for _ in range(30):
        o, status = with_status(q, k, v, sink, cu)
        assert status == 0
        if first is None:
            R.assert_close(o, ref, spread, err)
            first = o
        assert torch.equal(o, first)
    assert torch.equal(A.packed_attention(q, k, v, cu, sink), first)


@pytest.mark.parametrize("D", [64, 128])
def test_what_the_call_before_left_in_rows_that_no_load_writes(D):
    """Three heads to a key head fill 126 of a tile's 128 rows; the call before filled all of them, with NaN."""
    q, k, v, sink, cu = make([700, 300], 6, 2, D, seed=3)
    ref, spread, err = R.packed(q, k, v, cu, sink, 16, 8.0)
    before = make([256 * 80], 8, 2, D, seed=4)
    outs = []
    for value in (0.0, float("nan"), float("inf"), 3e38):
        A.packed_attention(before[0].fill_(value), *before[1:3], before[4])
        outs.append(A.packed_attention(q, k, v, cu, sink))
    R.assert_close(outs[0], ref, spread, err)
    assert all(torch.equal(o, outs[0]) for o in outs)
