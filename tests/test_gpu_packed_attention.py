"""Causal attention of packed sequences with grouped heads against its definition in 64 bits."""

import pytest
import torch

import algebraic_transformer_b200 as A
import ragged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(lens, H, Hkv, D, seed=0, start=0, tail=0, size=1.0, garbage=False):
    g = torch.Generator().manual_seed(seed)
    T = start + sum(lens) + tail
    q, k = (torch.randn((T, h, D), generator=g) for h in (H, Hkv))
    q, k = (size * t / t.square().mean(-1, keepdim=True).sqrt() for t in (q, k))
    v = torch.randn((T, Hkv, D), generator=g)
    if garbage:                                        # rows of no sequence hold anything
        for t in (q, k, v):
            t[:start] = float("nan")
            t[start + sum(lens):] = float("inf")
    sink = 0.7 * torch.randn(H, generator=g)
    return [t.bfloat16().to(DEV) for t in (q, k, v)] + [sink.to(DEV), R.lengths_to_cu(lens, start).to(DEV)]


def check(q, k, v, sink, cu, n=16, c=8.0):
    o = A.packed_attention(q, k, v, cu, sink, n=n, c=c)
    ref, spread, err = R.packed(q, k, v, cu, sink, n, c)
    R.assert_close(o, ref, spread, err)
    return o


LENS = [[1], [5, 1, 90], [128], [127, 129, 0, 1], [0, 0, 300], [513], [64, 0, 37, 255, 256, 257, 2]]


@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 64), (6, 2, 64), (4, 1, 128), (16, 2, 128)])
def test_lengths_and_groups(lens, H, Hkv, D):
    check(*make(lens, H, Hkv, D, seed=len(lens)))


@pytest.mark.parametrize("H,Hkv", [(5, 1), (7, 1), (24, 2), (48, 1), (128, 1)])
def test_odd_and_large_groups(H, Hkv):
    check(*make([33, 1, 70], H, Hkv, 64, seed=H))


@pytest.mark.parametrize("n", [2, 4, 8, 16, 32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [0.05, 1.0, 6.0])
def test_powers_and_score_sizes(n, D, size):
    q, k, v, sink, cu = make([200, 61], 3, 1, D, seed=n, size=size)
    check(q, k, v, sink, cu, n=n, c=8.0 if size < 2 else 3.0)
    check(q, k, v, None, cu, n=n, c=8.0 if size < 2 else 3.0)


def test_scores_far_outside_the_unshifted_range():
    """Rows whose scores are all very negative, all very large, and of both signs, beside ordinary ones."""
    q, k, v, sink, cu = make([300, 150], 4, 2, 64, seed=11)
    direction = torch.randn(64, generator=torch.Generator().manual_seed(1)).to(DEV)
    direction = (direction / direction.norm() * 8).bfloat16()
    k[:, 0] = (k[:, 0].float() * 0.5 + direction.float()).bfloat16()
    q[10:60, 0] = (-40 * direction.float()).bfloat16()           # x about -300: nothing but tiny weights
    q[60:90, 1] = (40 * direction.float()).bfloat16()
    q[200:230, 0] = (q[200:230, 0].float() * 50).bfloat16()
    q[310:312, 1] = 0
    for s in (sink, None, sink * 100, sink - 1000):
        check(q, k, v, s, cu)
        check(q, k, v, s, cu, n=32, c=1.0)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_no_sequence(D):
    q, k, v, sink, cu = make([77, 0, 130], 4, 2, D, seed=5, start=9, tail=140, garbage=True)
    o = check(q, k, v, sink, cu)
    assert (o[:9] == 0).all() and (o[9 + 207:] == 0).all()
    kept = torch.full_like(q, 3.0)
    got = A.packed_attention(q, k, v, cu, sink, out=kept)
    assert got is kept and (kept[:9] == 3).all() and (kept[216:] == 3).all() and torch.equal(kept[9:216], o[9:216])


def test_what_a_neighbour_holds_does_not_matter():
    q, k, v, sink, cu = make([70, 60, 200], 4, 2, 64, seed=6)
    want = A.packed_attention(q, k, v, cu, sink)
    for t, bad in ((k, float("nan")), (v, float("inf")), (v, float("nan")), (q, float("nan"))):
        t2 = t.clone()
        t2[70:130] = bad
        args = [t2 if x is t else x for x in (q, k, v)]
        got = A.packed_attention(*args, cu, sink)
        assert torch.equal(got[:70], want[:70]) and torch.equal(got[130:], want[130:])


def test_strides():
    """q, k, v side by side in one projection's output, o in a wider buffer, key heads ahead of tokens."""
    q, k, v, sink, cu = make([90, 40], 4, 2, 64, seed=8)
    want = A.packed_attention(q, k, v, cu, sink)
    T = q.shape[0]
    qkv = torch.cat([t.reshape(T, -1) for t in (q, k, v)], dim=1)
    wide = torch.zeros((T, 6, 64), dtype=torch.bfloat16, device=DEV)
    got = A.packed_attention(qkv[:, :256].view(T, 4, 64), qkv[:, 256:384].view(T, 2, 64), qkv[:, 384:].view(T, 2, 64), cu, sink,
                             out=wide[:, 1:5])
    assert torch.equal(got, want) and (wide[:, 0] == 0).all() and (wide[:, 5] == 0).all()
    ahead = k.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(A.packed_attention(q, ahead, v, cu, sink), want)


def test_few_long_sequences_are_cut_along_the_keys():
    q, k, v, sink, cu = make([2500, 700], 2, 1, 64, seed=9)
    check(q, k, v, sink, cu)
    q[2100:2200] *= 60                                             # parts with different references
    check(q, k, v, sink, cu)
    q, k, v, sink, cu = make([3001], 2, 2, 128, seed=10)
    check(q, k, v, None, cu)


def test_one_length_agrees_with_the_batched_operator():
    B, H, T, D = 3, 4, 200, 64
    q, k, v, sink, _ = make([B * T], H, H, D, seed=12)
    cu = R.lengths_to_cu([T] * B).to(DEV)
    batched = A.flash_attention(*(t.view(B, T, H, D).transpose(1, 2) for t in (q, k, v)), sink, kind="asinh", n=16, c=8.0,
                                range_guard=True, block=T)
    packed = A.packed_attention(q, k, v, cu, sink)
    a, b = batched.transpose(1, 2).reshape(B * T, H, D).double(), packed.double()
    assert float((a - b).norm() / a.norm()) < 2 * R.BF16           # each within BF16 of the weights' and of the result's rounding


def test_training_outputs():
    q, k, v, sink, cu = make([300, 0, 41, 129], 6, 2, 64, seed=13, tail=20, garbage=True)
    o, stat, rest = A.packed_attention(q, k, v, cu, sink, return_stat=True)
    ref, spread, err = R.packed(q, k, v, cu, sink, 16, 8.0)
    R.assert_close(o, ref, spread, err, weights=2.0 ** -16)
    rows = slice(0, 470)
    R.assert_close(o[rows].double() + rest[rows].double(), ref[rows], spread[rows], err, weights=2.0 ** -16, result=2.0 ** -16)
    # the statistic: p_sink = (rho(b / c) a)^n
    got = (R.rho(sink.double()[:, None].cpu() / 8) * stat[:, rows].double().cpu()) ** 16
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        for h in range(6):
            if b == a:
                continue
            x = q[a:b, h].double().cpu() @ k[a:b, h // 3].double().cpu().t() / (8 * 8.0)
            w = R.rho(x) ** 16
            w = w.tril().sum(1)
            s = R.rho(sink[h].double().cpu() / 8) ** 16
            assert float(((s / (s + w)) / got[h, a:b] - 1).abs().max()) < 2 * err + 16 * 2.0 ** -22


def test_graph_replayed_with_other_lengths_and_other_streams():
    q, k, v, sink, cu = make([300, 212], 4, 2, 64, seed=14)
    other = R.lengths_to_cu([100, 412]).to(DEV)
    want, want2 = A.packed_attention(q, k, v, cu, sink), A.packed_attention(q, k, v, other, sink)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    lens = cu.clone()
    with torch.cuda.stream(side):
        A.packed_attention(q, k, v, lens, sink)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = A.packed_attention(q, k, v, lens, sink)
    for cu_, w in ((cu, want), (other, want2), (cu, want)):
        lens.copy_(cu_)
        graph.replay()
        assert torch.equal(got, w)
    with torch.cuda.stream(side):
        outs = [A.packed_attention(q, k, v, x, sink) for x in (cu, other, cu)]
    here = [A.packed_attention(q, k, v, x, sink) for x in (other, cu, other)]
    torch.cuda.synchronize()
    for x, w in zip(outs + here, [want, want2, want, want2, want, want2]):
        assert torch.equal(x, w)


def test_lengths_that_lead_outside_are_clamped():
    q, k, v, sink, _ = make([100], 2, 1, 64, seed=15)
    for bad in ([0, 250], [-5, 60, 100], [50, 20, 100], [0, 2 ** 31 - 1], [100, 100], [90, -3]):
        o = A.packed_attention(q, k, v, torch.tensor(bad, dtype=torch.int32, device=DEV), sink)
        assert torch.isfinite(o.float()).all()
    want = A.packed_attention(q, k, v, torch.tensor([0, 100], dtype=torch.int32, device=DEV), sink)
    assert torch.equal(A.packed_attention(q, k, v, torch.tensor([0, 250], dtype=torch.int32, device=DEV), sink), want)


def test_nothing_to_do():
    q, k, v, sink, _ = make([40], 2, 1, 64, seed=16)
    o = A.packed_attention(q, k, v, torch.zeros(1, dtype=torch.int32, device=DEV), sink)
    assert (o == 0).all()
    o = A.packed_attention(q[:0], k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device=DEV), sink)
    assert o.shape == (0, 2, 64)
