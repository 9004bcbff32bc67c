"""The second pass over items whose values overflow the unshifted sum, at length: many items to a CTA, many calls, with the status word."""

import pytest
import torch

import algebraic_transformer_b200 as A
from algebraic_transformer_b200 import _lib as L
import ragged_reference as R
from test_gpu_packed_attention import make
from test_gpu_packed_paged_large_values import towards
from test_gpu_packed_short_items import with_status
from test_gpu_paged_attention import make as make_paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("count,H,Hkv,D", [(900, 6, 2, 64), (400, 4, 4, 128), (150, 2, 1, 64)])
@pytest.mark.parametrize("every", [1, 3])
def test_packed(count, H, Hkv, D, every):
    lens = [1 + (37 * i) % 300 for i in range(count)]
    q, k, v, sink, cu = make(lens, H, Hkv, D, seed=6, size=3.0)
    towards(q, k, D, 16)
    for a, b in list(zip(cu[:-1].tolist(), cu[1:].tolist()))[::every]:
        v[a:b] *= 2.0 ** 100
    first = None
    for _ in range(60):
        o, status = with_status(q, k, v, sink, cu)
        assert status == 0 and torch.isfinite(o).all()
        if first is None:
            some = torch.randperm(count, generator=torch.Generator().manual_seed(1))[:60].sort().values.tolist()
            for s in some:
                a, b = int(cu[s]), int(cu[s + 1])
                ref, spread, err = R.packed(q[a:b], k[a:b], v[a:b], torch.tensor([0, b - a]), sink, 16, 8.0)
                R.assert_close(o[a:b], ref, spread, err)
            first = o
        assert torch.equal(o, first)


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("H,Hkv,D", [(6, 2, 64), (12, 1, 128)])
def test_paged(H, Hkv, D, single):
    lib, S, page = L.load(), 500, 16
    lens = [1 + (53 * i) % 700 for i in range(S)]
    new = [1] * S if single else [min(n, 1 + (7 * i) % 50) for i, n in enumerate(lens)]
    a = make_paged(new, lens, H, Hkv, D, page, seed=7, size=3.0, garbage=False)
    q, kp, vp, table = a["q"], a["k_pages"], a["v_pages"], a["block_table"]
    towards(q, kp, D, 16)
    vp[::2] *= 2.0 ** 100
    o, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device=DEV)
    args = L.PagedAttnArgs(q=q.data_ptr(), k_pages=kp.data_ptr(), v_pages=vp.data_ptr(), o=o.data_ptr(), block_table=table.data_ptr(),
                           kv_lens=a["kv_lens"].data_ptr(), cu_seqlens=None if single else a["cu_seqlens"].data_ptr(), sink=a["sink_logit"].data_ptr(),
                           sequences=S, tokens=q.shape[0], H=H, Hkv=Hkv, D=D, pages=kp.shape[0], page_size=page, table_width=table.shape[1], n=16,
                           c=8.0, zero_tail=1, table_stride=table.stride(0), status=status.data_ptr(), q_stride=L.I64x2(*q.stride()[:2]),
                           o_stride=L.I64x2(*o.stride()[:2]), k_stride=L.I64x3(*kp.stride()[:3]), v_stride=L.I64x3(*vp.stride()[:3]))
    ws = torch.empty(lib.alg_paged_attn_workspace_bytes(args), dtype=torch.uint8, device=DEV)
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    first = None
    for _ in range(60):
        o.fill_(float("nan"))
        assert lib.alg_paged_attn_fwd(args, torch.cuda.current_stream().cuda_stream) == L.ALG_OK
        torch.cuda.synchronize()
        assert int(status) == 0 and torch.isfinite(o).all()
        if first is None:
            cu = a["cu_seqlens"].tolist()
            for s in torch.randperm(S, generator=torch.Generator().manual_seed(1))[:40].tolist():
                rows = slice(s, s + 1) if single else slice(cu[s], cu[s + 1])
                ref, spread, err = R.paged(q[rows], kp, vp, table[s:s + 1], lens[s:s + 1], torch.tensor([0, rows.stop - rows.start]),
                                           a["sink_logit"], 16, 8.0)
                R.assert_close(o[rows], ref, spread, err)
            first = o.clone()
        assert torch.equal(o, first)


def test_replayed_with_values_of_other_sizes():
    """One captured call, whose values need no second pass, then one, then none."""
    lens = [700, 3, 2300, 90]
    q, k, v, sink, cu = make(lens, 4, 2, 64, seed=8, size=3.0)
    paged = make_paged([20, 1, 60, 7], [400, 30, 2500, 9], 4, 2, 128, 32, seed=9, size=3.0, garbage=False)
    single = dict(make_paged([1] * 4, [400, 30, 2500, 9], 6, 2, 64, 16, seed=9, size=3.0, garbage=False), cu_seqlens=None)

    def calls():
        return (A.packed_attention(q, k, v, cu, sink), *A.packed_attention(q, k, v, cu, sink, return_stat=True), A.paged_attention(**paged),
                A.paged_attention(**single))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    values = [v, paged["v_pages"], single["v_pages"]]
    plain = [t.clone() for t in values]
    for scale in (1.0, 2.0 ** 100, 1.0, 2.0 ** 66):
        for t, p in zip(values, plain):
            t.copy_(p * scale)
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, calls()):
            assert torch.isfinite(got).all() and torch.equal(got, want)
