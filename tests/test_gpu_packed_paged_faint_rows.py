"""Rows whose keys weigh next to nothing beside the sink: the output is a faint mean of the values, but not zero."""

import pytest
import torch

import algebraic_transformer_b200 as A
import ragged_reference as R
from test_gpu_packed_attention import make
from test_gpu_paged_attention import make as make_paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def faint(q, k, x, D, c):
    """Every score is about x."""
    way = torch.randn(D, generator=torch.Generator().manual_seed(1))
    way = way / way.norm() * (abs(x) * D ** 0.5 * c) ** 0.5
    q[:] = (way * (1 if x > 0 else -1)).bfloat16().to(DEV)
    k[:] = way.bfloat16().to(DEV)


# (power, scores, the sinks' b / c): weights of 2^-80 to 2^-200 beside sinks of 2^-30 to 2^-64, as ratios no less than 2^-100
CASES = [(32, -6.9, -1.2), (32, -13.0, -1.8), (32, -20.0, -1.85), (16, -40.0, -7.5), (16, -100.0, -7.9), (8, -300.0, -7.9)]


@pytest.mark.parametrize("n,x,b", CASES)
@pytest.mark.parametrize("lens,H,Hkv,D", [([1, 5, 200, 1], 4, 2, 64), ([3, 140], 3, 1, 128), ([2500, 300], 2, 1, 64)], ids=["64", "128", "cut"])
def test_packed(lens, H, Hkv, D, n, x, b):
    q, k, v, sink, cu = make(lens, H, Hkv, D, seed=n)
    faint(q, k, x, D, 8.0)
    sink = torch.full_like(sink, 8.0 * b)
    ref, spread, err = R.packed(q, k, v, cu, sink, n, 8.0)
    assert float(spread.max()) > 2.0 ** -100
    o, stat, rest = A.packed_attention(q, k, v, cu, sink, n=n, return_stat=True)
    scale = 2.0 ** 90                                      # past the bound's absolute part
    for got, weights in ((A.packed_attention(q, k, v, cu, sink, n=n), R.BF16), (o, 2.0 ** -16)):
        R.assert_close(got.double() * scale, ref * scale, spread * scale, err, weights=weights)


@pytest.mark.parametrize("n,x,b", CASES)
@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_paged(D, single, n, x, b):
    lens = [1, 70, 900]
    a = make_paged([1, 1, 1] if single else [1, 20, 3], lens, 4, 2, D, 32, seed=n, garbage=False)
    faint(a["q"], a["k_pages"], x, D, 8.0)
    a["sink_logit"] = torch.full_like(a["sink_logit"], 8.0 * b)
    if single:
        a["cu_seqlens"] = None
    ref, spread, err = R.paged(a["q"], a["k_pages"], a["v_pages"], a["block_table"], lens, a["cu_seqlens"], a["sink_logit"], n, 8.0)
    scale = 2.0 ** 90
    R.assert_close(A.paged_attention(**a, n=n).double() * scale, ref * scale, spread * scale, err)
