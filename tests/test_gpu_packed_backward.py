"""Gradients of the attention over packed sequences against the formulas in 64 bits and against differences."""

import pytest
import torch

import algebraic_transformer_b200 as A
from algebraic_transformer_b200 import autograd as G
import ragged_reference as R
from test_gpu_packed_attention import LENS, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAMES = ("dq", "dk", "dv", "dsink")


def incoming(q, seed):
    return torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)


def gradients(q, k, v, sink, cu, d_o, n=16, c=8.0):
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)] + ([] if sink is None else [sink.detach().clone().requires_grad_()])
    o = G.packed_attention(*leaves[:3], cu, leaves[3] if sink is not None else None, n=n, c=c)
    return torch.autograd.grad(o, leaves, d_o)


def check(q, k, v, sink, cu, n=16, c=8.0, seed=100, d_o=None):
    d_o = incoming(q, seed) if d_o is None else d_o
    got = gradients(q, k, v, sink, cu, d_o, n, c)
    want, bound = R.packed_gradients(q, k, v, d_o, cu, sink, n, c)
    for name, g, w, b in zip(NAMES, got, want, bound):
        off = (g.double().cpu() - w).abs()
        assert torch.isfinite(g).all(), name
        worst = float((off / b).max())
        assert worst <= 1.0, f"{name}: {worst} times the bound"
    return got, want, bound


@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 64), (6, 2, 64), (4, 1, 128), (16, 2, 128)])
def test_lengths_and_groups(lens, H, Hkv, D):
    check(*make(lens, H, Hkv, D, seed=len(lens)))


@pytest.mark.parametrize("H,Hkv", [(5, 1), (24, 3), (48, 1)])
def test_odd_and_large_groups(H, Hkv):
    check(*make([33, 1, 170], H, Hkv, 64, seed=H))


@pytest.mark.parametrize("n", [2, 4, 8, 16, 32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [0.05, 1.0, 3.0])
def test_powers_and_score_sizes(n, D, size):
    q, k, v, sink, cu = make([200, 61], 3, 1, D, seed=n, size=size)
    check(q, k, v, sink, cu, n=n)
    check(q, k, v, None, cu, n=n)


def test_scores_far_outside_the_unshifted_range():
    q, k, v, sink, cu = make([300, 150], 4, 2, 64, seed=11)
    direction = torch.randn(64, generator=torch.Generator().manual_seed(1)).to(DEV)
    direction = (direction / direction.norm() * 8).bfloat16()
    k[:, 0] = (k[:, 0].float() * 0.5 + direction.float()).bfloat16()
    q[10:60, 0] = (-40 * direction.float()).bfloat16()
    q[60:90, 1] = (40 * direction.float()).bfloat16()
    q[200:230, 0] = (q[200:230, 0].float() * 20).bfloat16()
    for s in (sink, None, sink * 100):
        check(q, k, v, s, cu)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_no_sequence_have_no_gradient(D):
    q, k, v, sink, cu = make([77, 0, 130], 4, 2, D, seed=5, start=9, tail=140, garbage=True)
    d_o = incoming(q, 3)
    d_o[:9], d_o[216:] = float("nan"), float("inf")
    got, _, _ = check(q, k, v, sink, cu, d_o=d_o)
    for g in got[:3]:
        assert (g[:9] == 0).all() and (g[216:] == 0).all()


def test_what_a_neighbour_holds_does_not_matter():
    q, k, v, sink, cu = make([70, 60, 200], 4, 2, 64, seed=6)
    d_o = incoming(q, 4)
    want = gradients(q, k, v, sink, cu, d_o)
    for which in range(4):
        t = [q.clone(), k.clone(), v.clone(), d_o.clone()]
        t[which][70:130] = float("nan")
        got = gradients(*t[:3], sink, cu, t[3])
        for a, b in zip(got[:3], want[:3]):
            assert torch.equal(a[:70], b[:70]) and torch.equal(a[130:], b[130:])


def test_results_repeat():
    q, k, v, sink, cu = make([400, 1, 350, 90], 12, 4, 64, seed=7)
    d_o = incoming(q, 5)
    first = gradients(q, k, v, sink, cu, d_o)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, gradients(q, k, v, sink, cu, d_o)))


def test_against_differences():
    """Central differences of the definition in 64 bits, along random directions of each input."""
    q, k, v, sink, cu = make([40, 90], 4, 2, 64, seed=8)
    d_o = incoming(q, 6)
    got, _, bound = check(q, k, v, sink, cu, d_o=d_o)
    exact = [t.double().cpu() for t in (q, k, v)] + [sink.double().cpu()]

    def loss(x):
        o, _, _ = R.packed(*x[:3], cu, x[3], 16, 8.0)
        return float((o * d_o.double().cpu()).sum())

    for i in range(4):
        way = torch.randn(exact[i].shape, generator=torch.Generator().manual_seed(9 + i), dtype=torch.float64)
        step = 1e-5
        sides = [loss([x + s * step * way if j == i else x for j, x in enumerate(exact)]) for s in (1, -1)]
        slope = (sides[0] - sides[1]) / (2 * step)
        mine = float((got[i].double().cpu() * way).sum())
        assert abs(mine - slope) <= float((bound[i] * way.abs()).sum()) + 1e-6 * abs(slope) + 1e-7


def test_layouts_of_the_incoming_gradient():
    q, k, v, sink, cu = make([70, 50], 4, 2, 64, seed=9)
    d_o = incoming(q, 7)
    want = gradients(q, k, v, sink, cu, d_o)
    wide = torch.zeros((120, 6, 64), dtype=torch.bfloat16, device=DEV)
    wide[:, 1:5] = d_o
    ahead = d_o.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(120 * 256 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(120, 4, 64)
    odd.copy_(d_o)
    for other in (wide[:, 1:5], ahead, odd):
        assert all(torch.equal(a, b) for a, b in zip(want, gradients(q, k, v, sink, cu, other)))
    ones = gradients(q, k, v, sink, cu, torch.ones((), dtype=torch.bfloat16, device=DEV).expand(120, 4, 64))
    assert all(torch.equal(a, b) for a, b in zip(ones, gradients(q, k, v, sink, cu, torch.ones_like(q))))


def test_through_a_projection():
    """q, k and v as views of one projection's output: the gradient arrives there."""
    T, H, Hkv, D = 120, 4, 2, 64
    g = torch.Generator().manual_seed(10)
    qkv = torch.randn((T, (H + 2 * Hkv) * D), generator=g).bfloat16().to(DEV).requires_grad_()
    sink, cu = torch.zeros(H, device=DEV), R.lengths_to_cu([70, 50]).to(DEV)
    parts = lambda x: (x[:, : H * D].view(T, H, D), x[:, H * D: (H + Hkv) * D].view(T, Hkv, D), x[:, (H + Hkv) * D:].view(T, Hkv, D))  # noqa: E731
    o = G.packed_attention(*parts(qkv), cu, sink)
    d_o = incoming(o, 11)
    o.backward(d_o)
    want = gradients(*(p.detach().contiguous() for p in parts(qkv)), sink, cu, d_o)
    assert all(torch.equal(a, b) for a, b in zip(parts(qkv.grad), want[:3]))


def test_nothing_to_do():
    q, k, v, sink, _ = make([40], 2, 1, 64, seed=16)
    got = gradients(q, k, v, sink, torch.zeros(1, dtype=torch.int32, device=DEV), torch.ones_like(q))
    assert all((g == 0).all() for g in got)
    got = gradients(q[:0], k[:0], v[:0], sink, torch.zeros(3, dtype=torch.int32, device=DEV), q[:0])
    assert (got[3] == 0).all() and got[0].shape == (0, 2, 64)
