"""Waits that run out in the packed and paged operators: the status word says so, and no row of the outputs is left with a plausible
number that is not its result.  The kernels load only some of their tiles, and their waits last milliseconds."""

import pytest
import torch

import algebraic_transformer_b200 as A
from algebraic_transformer_b200 import _lib as L
from test_gpu_packed_attention import make
from test_gpu_paged_attention import make as make_paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BUDGET = 2_000_000


def stream():
    return torch.cuda.current_stream().cuda_stream


def result_or_nan(got, want):
    """Every row of the last axis is what it should be, or NaN; returns which are NaN."""
    nan = got.isnan().any(-1)
    assert bool((got.isnan().all(-1) == nan).all())
    assert torch.equal(got[~nan], want[~nan])
    return nan


def packed_args(q, k, v, sink, cu, o, stat, rest, status):
    lib, (T, H, D), Hkv = L.load(), q.shape, k.shape[1]
    a = L.PackedAttnArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=o.data_ptr(), cu_seqlens=cu.data_ptr(), sink=sink.data_ptr(),
                         stat=None if stat is None else stat.data_ptr(), o_rest=None if rest is None else rest.data_ptr(),
                         sequences=cu.numel() - 1, tokens=T, H=H, Hkv=Hkv, D=D, n=16, c=8.0, zero_tail=1, status=status.data_ptr())
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o)):
        setattr(a, name + "_stride", L.I64x2(*t.stride()[:2]))
    ws = torch.zeros(lib.alg_packed_attn_workspace_bytes(a), dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    return a, ws


# few items; more items of one tile than the CTAs take at once; items that are cut along the keys; three heads to a key head
SHAPES = [([300, 200], 4, 2, 64), ([1 + (37 * i) % 128 for i in range(900)], 4, 2, 64), ([2500, 700], 2, 1, 64), ([3001], 2, 2, 128), ([500, 90], 6, 2, 128)]


@pytest.mark.parametrize("max_loads", [0, 1, 2, 5, 12])
@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("lens,H,Hkv,D", SHAPES, ids=["few", "many", "cut64", "cut128", "three"])
def test_packed(lens, H, Hkv, D, train, max_loads):
    lib = L.load()
    q, k, v, sink, cu = make(lens, H, Hkv, D, seed=D, start=3, tail=5, garbage=True)
    want, want_stat, want_rest = A.packed_attention(q, k, v, cu, sink, return_stat=True)
    if not train:
        want = A.packed_attention(q, k, v, cu, sink)
    o, status = torch.full_like(q, 7.0), torch.zeros(1, dtype=torch.int32, device=DEV)
    stat, rest = (torch.full_like(want_stat, 7.0), torch.full_like(q, 7.0)) if train else (None, None)
    a, ws = packed_args(q, k, v, sink, cu, o, stat, rest, status)
    assert lib.alg_selftest_packed_timeout(a, max_loads, BUDGET, stream()) == L.ALG_OK
    torch.cuda.synchronize()
    rows = slice(3, 3 + sum(lens))
    nan = result_or_nan(o[rows], want[rows])
    assert int(status) == int(bool(nan.any())) and (max_loads > 1 or bool(nan.all()))      # few items of few tiles may have all they need
    assert bool((o[:3] == 0).all()) and bool((o[rows.stop:] == 0).all())
    if train:
        assert torch.equal(result_or_nan(rest[rows], want_rest[rows]), nan)
        got = stat[:, rows].t()
        assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], want_stat[:, rows].t()[~nan])
    status.zero_()
    assert lib.alg_packed_attn_fwd(a, stream()) == L.ALG_OK
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(o[rows], want[rows])


@pytest.mark.parametrize("max_loads", [0, 1, 3])
@pytest.mark.parametrize("with_sink", [True, False])
@pytest.mark.parametrize("lens,H,Hkv,D", [([300, 200], 4, 2, 64), ([500, 90], 6, 2, 128), ([10] * 300, 2, 2, 64)], ids=["64", "128", "short"])
def test_packed_backward(lens, H, Hkv, D, with_sink, max_loads):
    lib = L.load()
    q, k, v, sink, cu = make(lens, H, Hkv, D, seed=1 + D, tail=5)
    sink = sink if with_sink else None
    d_o = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    o, stat, rest = A.packed_attention(q, k, v, cu, sink, return_stat=True)
    want = A.packed_attention_backward(q, k, v, o, d_o, stat, rest, cu, sink)
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    dsink, status = torch.full((H,), 7.0, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    a = L.PackedAttnBwdArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=o.data_ptr(), o_rest=rest.data_ptr(), d_o=d_o.data_ptr(),
                            stat=stat.data_ptr(), cu_seqlens=cu.data_ptr(), sink=sink.data_ptr() if with_sink else None, dq=grads[0].data_ptr(),
                            dk=grads[1].data_ptr(), dv=grads[2].data_ptr(), dsink=dsink.data_ptr() if with_sink else None, sequences=cu.numel() - 1,
                            tokens=q.shape[0], H=H, Hkv=Hkv, D=D, n=16, c=8.0, status=status.data_ptr())
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o), ("do", d_o), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        setattr(a, name + "_stride", L.I64x2(*t.stride()[:2]))
    ws = torch.zeros(lib.alg_packed_attn_bwd_workspace_bytes(a), dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    assert lib.alg_selftest_packed_bwd_timeout(a, max_loads, BUDGET, stream()) == L.ALG_OK
    torch.cuda.synchronize()
    short = max_loads >= -(-max(lens) // 64) * (H // Hkv)           # then every block has all of its tiles
    assert int(status) == (0 if short else 1)
    n = sum(lens)
    for g, w in zip(grads, want):
        nan = result_or_nan(g[:n], w[:n])
        assert bool((g[n:] == 0).all()) and (max_loads > 0 or bool(nan.all()))
        assert not short or not bool(nan.any())
    if with_sink and not short:
        assert bool((dsink.isnan()).all())
    status.zero_()
    assert lib.alg_packed_attn_bwd(a, stream()) == L.ALG_OK
    torch.cuda.synchronize()
    assert int(status) == 0 and all(torch.equal(g, w) for g, w in zip(grads, want)) and (not with_sink or torch.equal(dsink, want[3]))


@pytest.mark.parametrize("max_loads", [0, 1, 4])
@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("lens,H,Hkv,D,page", [([400, 90, 1000], 4, 2, 64, 16), ([5000, 2100], 16, 1, 128, 64), ([200] * 300, 2, 1, 64, 32)],
                         ids=["few", "long", "many"])
def test_paged(lens, H, Hkv, D, page, single, max_loads):
    lib, S = L.load(), len(lens)
    new = [1] * S if single else [1 + (7 * i) % 40 for i in range(S)]
    a = make_paged(new, lens, H, Hkv, D, page, seed=D)
    if single:
        a["cu_seqlens"] = None
    want = A.paged_attention(**a)
    q, kp, vp, table = a["q"], a["k_pages"], a["v_pages"], a["block_table"]
    o, status = torch.full_like(q, 7.0), torch.zeros(1, dtype=torch.int32, device=DEV)
    args = L.PagedAttnArgs(q=q.data_ptr(), k_pages=kp.data_ptr(), v_pages=vp.data_ptr(), o=o.data_ptr(), block_table=table.data_ptr(),
                           kv_lens=a["kv_lens"].data_ptr(), cu_seqlens=None if single else a["cu_seqlens"].data_ptr(),
                           sink=a["sink_logit"].data_ptr(), sequences=S, tokens=q.shape[0], H=H, Hkv=Hkv, D=D, pages=kp.shape[0], page_size=page,
                           table_width=table.shape[1], n=16, c=8.0, zero_tail=1, table_stride=table.stride(0), status=status.data_ptr(),
                           q_stride=L.I64x2(*q.stride()[:2]), o_stride=L.I64x2(*o.stride()[:2]), k_stride=L.I64x3(*kp.stride()[:3]),
                           v_stride=L.I64x3(*vp.stride()[:3]))
    ws = torch.zeros(lib.alg_paged_attn_workspace_bytes(args), dtype=torch.uint8, device=DEV)
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    assert lib.alg_selftest_paged_timeout(args, max_loads, BUDGET, stream()) == L.ALG_OK
    torch.cuda.synchronize()
    nan = result_or_nan(o, want)
    assert int(status) == int(bool(nan.any())) and (max_loads > 0 or bool(nan.all()))
    status.zero_()
    assert lib.alg_paged_attn_fwd(args, stream()) == L.ALG_OK
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(o, want)


def test_refusals():
    lib = L.load()
    q, k, v, sink, cu = make([40], 2, 1, 64)
    o, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device=DEV)
    a, ws = packed_args(q, k, v, sink, cu, o, None, None, status)
    assert lib.alg_selftest_packed_timeout(a, 1, 5_000_000_000, stream()) == L.ALG_ERR_INVALID
    assert lib.alg_selftest_packed_timeout(a, 1, 0, stream()) == L.ALG_ERR_INVALID
    assert lib.alg_selftest_packed_timeout(a, -1, BUDGET, stream()) == L.ALG_ERR_INVALID
    a.status = None
    assert lib.alg_selftest_packed_timeout(a, 1, BUDGET, stream()) == L.ALG_ERR_INVALID
    for fn in (lib.alg_selftest_packed_timeout, lib.alg_selftest_packed_bwd_timeout, lib.alg_selftest_paged_timeout):
        assert fn(None, 1, BUDGET, stream()) == L.ALG_ERR_INVALID
