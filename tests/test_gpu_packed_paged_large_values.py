"""Values of any size: unshifted weights go up to 2^64, so that values far inside the type's range would take their sum out of fp32's.
The result is a mean of the values and has to come out finite as long as the sum of a row's visible |v| is."""

import pytest
import torch

import algebraic_transformer_b200 as A
import ragged_reference as R
from test_gpu_packed_attention import make
from test_gpu_paged_attention import make as make_paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# (n, scale of the rows): scores up to near the end of the unshifted range, which is x = 7.97, 8 and 1.875 at n = 16, 4 and 32
POWERS = [(16, 3.0), (4, 3.0), (32, 1.2)]


def towards(q, k, D, n):
    """Some queries and keys in one direction: scores close to the end of the range, and beyond it."""
    way = torch.randn(D, generator=torch.Generator().manual_seed(1))
    way = way / way.norm() * {16: 7.9, 4: 7.9, 32: 1.85}[n] ** 0.5 * (D ** 0.5 * 8.0) ** 0.5
    q[5::7, :] = way.bfloat16().to(DEV)
    k.view(-1, k.shape[-2], D)[3::11] = way.bfloat16().to(DEV)


def sized(v, kind):
    if kind == "one":                                     # a few large values among ordinary ones
        v = v.clone()
        v.view(-1, v.shape[-2], v.shape[-1])[4::50, :, 3::16] *= 2.0 ** 80
        return v
    return (v.float() * kind).bfloat16()


SIZES = ["one", 2.0 ** 66, 2.0 ** 100, 2.0 ** 112, 2.0 ** -40]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("n,rows", POWERS)
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (3, 1, 128)])
def test_packed(H, Hkv, D, n, rows, size):
    q, k, v, sink, cu = make([300, 1, 90, 400], H, Hkv, D, seed=n, size=rows)
    towards(q, k, D, n)
    v = sized(v, size)
    for s in (sink, None):
        ref, spread, err = R.packed(q, k, v, cu, s, n, 8.0)
        R.assert_close(A.packed_attention(q, k, v, cu, s, n=n), ref, spread, err)
        o, stat, rest = A.packed_attention(q, k, v, cu, s, n=n, return_stat=True)
        R.assert_close(o, ref, spread, err, weights=2.0 ** -16)
        R.assert_close(o.double() + rest.double(), ref, spread, err, weights=2.0 ** -16, result=2.0 ** -16)


@pytest.mark.parametrize("size", ["one", 2.0 ** 66, 2.0 ** 100])
@pytest.mark.parametrize("D", [64, 128])
def test_packed_gradients(D, size):
    q, k, v, sink, cu = make([300, 1, 90], 4, 2, D, seed=3, size=3.0)
    towards(q, k, D, 16)
    v = sized(v, size)
    d_o = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    o, stat, rest = A.packed_attention(q, k, v, cu, sink, return_stat=True)
    got = A.packed_attention_backward(q, k, v, o, d_o, stat, rest, cu, sink)
    want, bound = R.packed_gradients(q, k, v, d_o, cu, sink, 16, 8.0)
    for g, w, b in zip(got, want, bound):
        assert torch.isfinite(g).all() and float(((g.double().cpu() - w).abs() / b).max()) <= 1.0


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("D", [64, 128])
def test_packed_cut_along_the_keys(D, size):
    q, k, v, sink, cu = make([3001, 300], 2, 1, D, seed=4, size=3.0)
    towards(q, k, D, 16)
    v = sized(v, size)
    for s in (sink, None):
        R.assert_close(A.packed_attention(q, k, v, cu, s), *R.packed(q, k, v, cu, s, 16, 8.0))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("n,rows", POWERS)
@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (12, 1, 64), (3, 1, 128), (24, 1, 128)])
def test_paged(H, Hkv, D, single, n, rows, size):
    lens = [700, 1, 60, 2500]
    a = make_paged([1] * 4 if single else [40, 1, 9, 3], lens, H, Hkv, D, 32, seed=n, size=rows, garbage=False)
    a["q"], a["k_pages"] = a["q"].clone(), a["k_pages"].clone()
    towards(a["q"], a["k_pages"], D, n)
    a["v_pages"] = sized(a["v_pages"], size)
    if single:
        a["cu_seqlens"] = None
        a["q"][3] = a["q"][0]
    for s in (a["sink_logit"], None):
        o = A.paged_attention(**dict(a, sink_logit=s), n=n)
        R.assert_close(o, *R.paged(a["q"], a["k_pages"], a["v_pages"], a["block_table"], lens, a["cu_seqlens"], s, n, 8.0))


@pytest.mark.parametrize("D", [64, 128])
def test_rows_beside_a_large_value_keep_their_bits(D):
    """A row that is weighed again for its values leaves the others as they were."""
    q, k, v, sink, cu = make([700, 60], 4, 2, D, seed=5, size=3.0)
    want = A.packed_attention(q, k, v, cu, sink)
    large = v.clone()
    large[650, 1, 7] = 3e38                               # seen by the last 50 tokens of the first sequence, heads 2 and 3
    got = A.packed_attention(q, k, large, cu, sink)
    assert torch.equal(got[:650], want[:650]) and torch.equal(got[700:], want[700:]) and torch.equal(got[:, :2], want[:, :2])
    a = make_paged([1, 1], [700, 60], 4, 2, D, 32, seed=5, size=3.0, garbage=False)
    a["cu_seqlens"] = None
    want = A.paged_attention(**a)
    a["v_pages"] = a["v_pages"].clone()
    a["v_pages"][int(a["block_table"][0, 20]), 3, 1, 7] = 3e38
    got = A.paged_attention(**a)
    assert torch.equal(got[1], want[1]) and torch.equal(got[:, :2], want[:, :2]) and torch.isfinite(got.float()).all()


def test_many_items_are_weighed_again():
    """More items to a CTA than it holds at a time, all of which, or every third of which, overflow."""
    lens = [1 + (37 * i) % 128 for i in range(900)]
    q, k, v, sink, cu = make(lens, 6, 2, 64, seed=6, size=3.0)
    towards(q, k, 64, 16)
    for some in (slice(None), slice(0, None, 3)):
        large = v.clone()
        for a, b in list(zip(cu[:-1].tolist(), cu[1:].tolist()))[some]:
            large[a:b] *= 2.0 ** 100
        o = A.packed_attention(q, k, large, cu, sink)
        ref, spread, err = R.packed(q, k, large, cu, sink, 16, 8.0)
        R.assert_close(o, ref, spread, err)
        for _ in range(5):
            assert torch.equal(A.packed_attention(q, k, large, cu, sink), o)
