"""Offsets that decrease: every sequence stays within the rows from the first offset to the last, so that keys whose norms are taken are
all that it meets, and rows outside are nobody's."""

import pytest
import torch

import algebraic_transformer_b200 as A
import ragged_reference as R
from test_gpu_packed_attention import make
from test_gpu_paged_attention import make as make_paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = 400
# the offsets as they are given, and what they come to: each end within the first and the last offset, an end ahead of its start an empty
# sequence.  The last but one gives its five rows to two sequences.
DECREASING = [([200, 60, 400], [(200, 200), (200, 400)]), ([50, 20, 100, 350], [(50, 50), (50, 100), (100, 350)]),
              ([300, 10, 250, 390], [(300, 300), (300, 300), (300, 390)]), ([390, 500, -7, 395], [(390, 395), (395, 395), (390, 395)]),
              ([120, 0], [(120, 120)])]


def offsets(cu):
    return torch.tensor(cu, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("given,meant", DECREASING)
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (3, 1, 128)])
def test_packed(given, meant, H, Hkv, D):
    """Keys outside the extent are large: weights that went unshifted by the norms of those inside would leave the range."""
    q, k, v, sink, _ = make([T], H, Hkv, D, seed=D)
    inside = torch.zeros(T, dtype=torch.bool, device=DEV)
    for a, b in meant:
        inside[a:b] = True
    k[~inside] = (k[~inside].float() * 3000).bfloat16()
    for s in (sink, None):
        o = A.packed_attention(q, k, v, offsets(given), s)
        for a, b in meant:
            ref, spread, err = R.packed(q, k, v, torch.tensor([a, b]), s, 16, 8.0)
            R.assert_close(o[a:b], ref[a:b], spread[a:b], err)
        assert bool((o[~inside] == 0).all())
        kept = torch.full_like(q, 3.0)
        A.packed_attention(q, k, v, offsets(given), s, out=kept)
        assert bool((kept[~inside] == 3).all()) and torch.equal(kept[inside], o[inside])


@pytest.mark.parametrize("given,meant", DECREASING)
def test_packed_gradients(given, meant):
    q, k, v, sink, _ = make([T], 4, 2, 64, seed=1)
    d_o = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    o, stat, rest = A.packed_attention(q, k, v, offsets(given), sink, return_stat=True)
    got = A.packed_attention_backward(q, k, v, o, d_o, stat, rest, offsets(given), sink)
    each = [R.packed_gradients(q, k, v, d_o, torch.tensor(rows), sink, 16, 8.0) for rows in meant]
    outside = torch.ones(T, dtype=torch.bool)
    for (a, b), (want, bound) in zip(meant, each):
        outside[a:b] = False
        for g, w, e in zip(got[:3], want, bound):
            assert bool(((g.double().cpu() - w).abs() <= e)[a:b].all())
    assert all(bool((g.cpu()[outside] == 0).all()) for g in got[:3])
    sums = [sum(pair[i][3] for pair in each) for i in range(2)]      # a sink's gradient is over all sequences
    assert bool(((got[3].double().cpu() - sums[0]).abs() <= sums[1]).all())


@pytest.mark.parametrize("given,meant", DECREASING)
def test_paged_chunks(given, meant):
    lens = [b - a + 30 for a, b in meant]
    q = make([T], 4, 2, 64, seed=4)[0]
    a = make_paged([1] * len(lens), lens, 4, 2, 64, 32, seed=5, garbage=False)
    o = A.paged_attention(**dict(a, q=q, cu_seqlens=offsets(given)))
    outside = torch.ones(T, dtype=torch.bool, device=DEV)
    for i, (first, end) in enumerate(meant):
        ref, spread, err = R.paged(q[first:end], a["k_pages"], a["v_pages"], a["block_table"][i:i + 1], lens[i:i + 1],
                                   torch.tensor([0, end - first]), a["sink_logit"], 16, 8.0)
        if sum(f < end and first < e for f, e in meant) == 1:        # else the other sequence may have written the rows
            R.assert_close(o[first:end], ref, spread, err)
        outside[first:end] = False
    assert torch.isfinite(o.float()).all() and bool((o[outside] == 0).all())


@pytest.mark.parametrize("given", [given for given, _ in DECREASING])
def test_append_stays_in_the_pages(given):
    """Which sequence a token counts to is open; it is written to that sequence's pages or not at all."""
    lens = [100] * (len(given) - 1)
    q, k, v, _, _ = make([T], 4, 2, 64, seed=4)
    a = make_paged([1] * len(lens), lens, 4, 2, 64, 32, seed=5, garbage=False)
    pages = [a["k_pages"].clone(), a["v_pages"].clone()]
    angle = torch.rand((a["block_table"].shape[1] * 32, 32), generator=torch.Generator().manual_seed(6)).to(DEV)
    o = A.paged_append(q, k, v, *pages, a["block_table"], a["kv_lens"], angle.cos(), angle.sin(), offsets(given))
    assert torch.isfinite(o.float()).all()
    unused = torch.ones(pages[0].shape[0], dtype=torch.bool, device=DEV)
    unused[a["block_table"].long().flatten()] = False
    assert torch.equal(pages[0][unused], a["k_pages"][unused]) and torch.equal(pages[1][unused], a["v_pages"][unused])
