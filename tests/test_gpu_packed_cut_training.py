"""Training over sequences long enough to be cut along the keys: the statistic and the output's second half then come from the kernel that adds
the parts up, and every gradient depends on them."""

import pytest
import torch

import algebraic_transformer_b200 as A
from algebraic_transformer_b200 import autograd as G
import ragged_reference as R
from test_gpu_packed_attention import make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CASES = [([2500, 700], 2, 1, 64), ([3001], 2, 2, 128), ([2200, 5, 2300], 3, 1, 64)]


@pytest.mark.parametrize("with_sink", [True, False])
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("lens,H,Hkv,D", CASES, ids=["64", "128", "three"])
def test_outputs_and_gradients(lens, H, Hkv, D, apart, with_sink):
    q, k, v, sink, cu = make(lens, H, Hkv, D, seed=D)
    if apart:                                                      # parts of a row with different references
        q[2100:2180] = (q[2100:2180].float() * 20).bfloat16()
    sink = sink if with_sink else None
    d_o = torch.randn(q.shape, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    o, stat, rest = A.packed_attention(q, k, v, cu, sink, return_stat=True)
    ref, spread, err = R.packed(q, k, v, cu, sink, 16, 8.0)
    R.assert_close(o, ref, spread, err, weights=2.0 ** -16)
    R.assert_close(o.double() + rest.double(), ref, spread, err, weights=2.0 ** -16, result=2.0 ** -16)
    # the statistic: p of a row's own key is (rho(x) a)^n; relative error: that of the weights, once in the sum and once in the power, and the root's
    at = torch.arange(q.shape[0])
    x = (q.double().cpu() * k.double().cpu().repeat_interleave(H // Hkv, dim=1)).sum(-1) / (D ** 0.5 * 8.0)
    got = 16 * (torch.asinh(x) + stat.double().cpu().t().log())
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        rows = torch.unique(torch.cat([torch.arange(a, b, 97), torch.arange(max(a, b - 3), b)])).clamp(max=b - 1)
        rows = rows[(rows >= a) & (rows < b)]
        for h in range(H):
            s = q[rows, h].double().cpu() @ k[a:b, h // (H // Hkv)].double().cpu().t() / (D ** 0.5 * 8.0)
            logw = (16 * torch.asinh(s)).masked_fill(at[a:b][None] > rows[:, None], -float("inf"))
            if with_sink:
                logw = torch.cat([logw, (16 * torch.asinh(sink[h].double().cpu() / 8)).expand(len(rows), 1)], dim=1)
            want = 16 * torch.asinh(x[rows, h]) - logw.logsumexp(dim=1)
            assert float((got[rows, h] - want).abs().max()) < 2 * err + 16 * 2.0 ** -21
    grads = A.packed_attention_backward(q, k, v, o, d_o, stat, rest, cu, sink)
    want, bound = R.packed_gradients(q, k, v, d_o, cu, sink, 16, 8.0)
    for name, g, w, b in zip(("dq", "dk", "dv", "dsink"), grads, want, bound):
        if g is not None:
            assert torch.isfinite(g).all() and float(((g.double().cpu() - w).abs() / b).max()) <= 1.0, name


def test_repeats_and_agrees_with_autograd():
    q, k, v, sink, cu = make([2500, 700], 2, 1, 64, seed=3)
    d_o = torch.randn(q.shape, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    o, stat, rest = A.packed_attention(q, k, v, cu, sink, return_stat=True)
    want = A.packed_attention_backward(q, k, v, o, d_o, stat, rest, cu, sink)
    for _ in range(3):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, sink)]
        out = G.packed_attention(*leaves[:3], cu, leaves[3])
        assert torch.equal(out, o)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, d_o), want))
