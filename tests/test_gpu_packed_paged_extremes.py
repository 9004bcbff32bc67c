"""The packed and paged operators at the ends of what their arguments may hold: infinite and lowest sinks, rows whose squares leave the
range, sequences that outgrow their table, more sequences than a plan's threads, an offset past 32 bits, calls side by side."""

import pytest
import torch

import algebraic_transformer_b200 as A
from algebraic_transformer_b200 import autograd as G
import ragged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, LOWEST = float("inf"), torch.finfo(torch.float32).min


def normal(*shape, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * size).to(torch.bfloat16).to(DEV)


def pages_of(lens, Hkv, D, page, seed=5):
    width = max(1, -(-max(lens) // page))
    count = len(lens) * width + 3
    table = torch.randperm(count, generator=torch.Generator().manual_seed(seed))[: len(lens) * width].reshape(len(lens), width)
    return normal(count, page, Hkv, D, seed=seed + 1), normal(count, page, Hkv, D, seed=seed + 2), table.to(torch.int32).to(DEV)


@pytest.mark.parametrize("T", [40, 700])
@pytest.mark.parametrize("D", [64, 128])
def test_sinks_without_bounds(T, D):
    """A sink of -inf, or of the type's lowest value, takes no weight; one of +inf takes all."""
    q, k, v, d_o = normal(T, 4, D), normal(T, 2, D, seed=1), normal(T, 2, D, seed=2), normal(T, 4, D, seed=3)
    cu = R.lengths_to_cu([T]).to(DEV)
    sink = torch.tensor([-INF, 0.5, LOWEST, 3.0], device=DEV)
    o, stat, rest = A.packed_attention(q, k, v, cu, sink, return_stat=True)
    R.assert_close(A.packed_attention(q, k, v, cu, sink), *R.packed(q, k, v, cu.cpu(), sink, 16, 8.0))
    got = A.packed_attention_backward(q, k, v, o, d_o, stat, rest, cu, sink)
    want, bound = R.packed_gradients(q, k, v, d_o, cu.cpu(), sink, 16, 8.0)
    for a, b, e in zip(got, want, bound):
        assert bool(((a.double().cpu() - b).abs() <= e).all())
    everything = torch.full((4,), INF, device=DEV)
    o, stat, rest = A.packed_attention(q, k, v, cu, everything, return_stat=True)
    for t in (A.packed_attention(q, k, v, cu, everything), o, *A.packed_attention_backward(q, k, v, o, d_o, stat, rest, cu, everything)):
        assert bool((t == 0).all())


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("lens", [[5, 0, 300], [6000]])
def test_sinks_without_bounds_over_pages(single, lens):
    kp, vp, table = pages_of(lens, 2, 64, 32)
    new = [1] * len(lens) if single else [2] * len(lens)
    cu, kv = R.lengths_to_cu(new), torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = normal(sum(new), 4, 64)
    sink = torch.tensor([-INF, 0.5, LOWEST, 3.0], device=DEV)
    got = A.paged_attention(q, kp, vp, table, kv, None if single else cu.to(DEV), sink)
    R.assert_close(got, *R.paged(q, kp, vp, table, lens, cu, sink, 16, 8.0))
    assert bool((A.paged_attention(q, kp, vp, table, kv, None if single else cu.to(DEV), torch.full((4,), INF, device=DEV)) == 0).all())
    nan = A.paged_attention(q, kp, vp, table, kv, None if single else cu.to(DEV), torch.tensor([0.0, float("nan"), 0.0, 0.0], device=DEV))
    has_keys = torch.tensor([n > 0 for n, m in zip(lens, new) for _ in range(m)])
    assert bool(nan[has_keys][:, 1].isnan().all()) and not bool(nan[:, [0, 2, 3]].isnan().any())


@pytest.mark.parametrize("tiny_keys", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_whose_squares_leave_the_range(tiny_keys, D):
    """|q| near 2^80 and |k| near 2^-78, or the other way round: neither squared norm is a float32, and the scores are far out of the
    range of the unshifted weights."""
    T = 400
    up, down = 2.0 ** 80, 2.0 ** -78
    q = (normal(T, 2, D).float() * (up if tiny_keys else down)).to(torch.bfloat16)
    k = (normal(T, 1, D, seed=1).float() * (down if tiny_keys else up)).to(torch.bfloat16)
    v, cu = normal(T, 1, D, seed=2), R.lengths_to_cu([T - 10, 10])
    R.assert_close(A.packed_attention(q, k, v, cu.to(DEV), c=0.0625), *R.packed(q, k, v, cu, None, 16, 0.0625))


@pytest.mark.parametrize("given", [False, True])
def test_tokens_behind_the_end_of_the_table(given):
    """A sequence that outgrows its table loses its newest tokens, not a key that stands there."""
    page, D, Hkv, H = 16, 64, 2, 4
    kp, vp, table = pages_of([32, 32, 32], Hkv, D, page)
    before = kp.clone(), vp.clone()
    cu, kv = R.lengths_to_cu([4, 1, 2]), torch.tensor([35, 2 ** 31 - 1, 32], dtype=torch.int32, device=DEV)
    q, k, v = normal(7, H, D), normal(7, Hkv, D, seed=1), normal(7, Hkv, D, seed=2)
    angle = torch.arange(32)[:, None] * torch.rand(D // 2, generator=torch.Generator().manual_seed(1))[None]
    cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)
    out = torch.full_like(q, 7.0) if given else None
    o = A.paged_append(q, k, v, kp, vp, table, kv, cos, sin, cu.to(DEV), out=out)
    lost = [1, 2, 3, 4]
    assert bool((o[lost] == (7.0 if given else 0.0)).all())
    # the tokens that have a place: token 0 at position 31 of sequence 0, tokens 5 and 6 at 30 and 31 of sequence 2
    for token, s, at in ((0, 0, 31), (5, 2, 30), (6, 2, 31)):
        number = int(table[s, at // page])
        assert torch.equal(vp[number, at % page], v[token])
        before[0][number, at % page] = kp[number, at % page]
        before[1][number, at % page] = v[token]
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])


def test_more_sequences_than_the_plan_has_threads():
    lens = [(7 * i) % 5 for i in range(2500)]
    T = sum(lens)
    q, k, v, d_o = normal(T, 2, 64), normal(T, 1, 64, seed=1), normal(T, 1, 64, seed=2), normal(T, 2, 64, seed=3)
    cu = R.lengths_to_cu(lens)
    R.assert_close(A.packed_attention(q, k, v, cu.to(DEV)), *R.packed(q, k, v, cu, None, 16, 8.0))
    o, stat, rest = A.packed_attention(q, k, v, cu.to(DEV), return_stat=True)
    got = A.packed_attention_backward(q, k, v, o, d_o, stat, rest, cu.to(DEV))
    want, bound = R.packed_gradients(q, k, v, d_o, cu, None, 16, 8.0)
    for a, b, e in zip(got[:3], want, bound):
        assert bool(((a.double().cpu() - b).abs() <= e).all())


@pytest.mark.parametrize("single", [False, True])
def test_more_sequences_than_threads_over_pages(single):
    lens = [1 + (11 * i) % 40 for i in range(1500)]
    kp, vp, table = pages_of(lens, 1, 64, 16)
    q, kv = normal(len(lens), 2, 64), torch.tensor(lens, dtype=torch.int32, device=DEV)
    cu = R.lengths_to_cu([1] * len(lens))
    got = A.paged_attention(q, kp, vp, table, kv, None if single else cu.to(DEV))
    R.assert_close(got, *R.paged(q, kp, vp, table, lens, cu, None, 16, 8.0))


@pytest.mark.parametrize("single", [False, True])
def test_pages_past_32_bits_of_offset(single):
    """A pool of 2^31 elements and more to each of K and V (strided over one allocation of 8.7 GB): its last pages."""
    page, Hkv, D = 32, 2, 64
    stride = 1 << 21                                        # elements from page to page
    count = 1040
    pool = torch.empty((count, 2, stride // 2), dtype=torch.bfloat16, device=DEV)
    kp = pool[:, 0, : page * Hkv * D].view(count, page, Hkv, D)
    vp = pool[:, 1, : page * Hkv * D].view(count, page, Hkv, D)
    assert kp.stride(0) * (count - 1) > 2 ** 31
    table = torch.tensor([[1039, 3], [1030, 1027]], dtype=torch.int32, device=DEV)
    lens = [50, 33]
    kp[table.long().flatten()] = normal(4, page, Hkv, D, seed=4)
    vp[table.long().flatten()] = normal(4, page, Hkv, D, seed=5)
    new = [1, 1] if single else [3, 1]
    cu, kv = R.lengths_to_cu(new), torch.tensor(lens, dtype=torch.int32, device=DEV)
    q, k, v = normal(sum(new), 4, D), normal(sum(new), Hkv, D, seed=1), normal(sum(new), Hkv, D, seed=2)
    cos, sin = torch.ones((64, D // 2), device=DEV), torch.zeros((64, D // 2), device=DEV)
    q2 = A.paged_append(q, k, v, kp, vp, table, kv, cos, sin, None if single else cu.to(DEV))
    assert torch.equal(vp[1027, 0], v[-1])
    small = torch.unique(table.flatten())
    index = torch.searchsorted(small, table)
    o, spread, err = R.paged(q2, kp[small.long()], vp[small.long()], index, lens, cu, None, 16, 8.0)
    R.assert_close(A.paged_attention(q2, kp, vp, table, kv, None if single else cu.to(DEV)), o, spread, err)


def test_calls_side_by_side():
    """Two streams, each with a chain of append and attention over a cache of its own, against the same chains one after the other."""
    def chain(i, out):
        lens = [40 + i, 900 + i, 3]
        kp, vp, table = pages_of([n + 8 for n in lens], 2, 128, 64, seed=10 * i)
        cos, sin = torch.ones((table.shape[1] * 64, 64), device=DEV), torch.zeros((table.shape[1] * 64, 64), device=DEV)
        inputs = [(normal(3, 8, 128, seed=100 * i + t), normal(3, 2, 128, seed=200 * i + t)) for t in range(8)]
        counts = [torch.tensor([n + t + 1 for n in lens], dtype=torch.int32, device=DEV) for t in range(8)]
        torch.cuda.synchronize()
        def run():
            for t, (q, k) in enumerate(inputs):
                q2 = A.paged_append(q, k, k, kp, vp, table, counts[t], cos, sin)
                out.append(A.paged_attention(q2, kp, vp, table, counts[t]))
        return run
    alone, beside = ([], []), ([], [])
    for i in range(2):
        chain(i + 1, alone[i])()
    torch.cuda.synchronize()
    runs = [chain(i + 1, beside[i]) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for run, stream in zip(runs, streams):
        with torch.cuda.stream(stream):
            run()
    torch.cuda.synchronize()
    for a, b in zip(alone, beside):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_captured_training_step():
    """Forward and backward in one graph, replayed with other lengths and values."""
    T, H, Hkv, D = 500, 4, 2, 64
    q, k, v, d_o = normal(T, H, D), normal(T, Hkv, D, seed=1), normal(T, Hkv, D, seed=2), normal(T, H, D, seed=3)
    sink, cu = torch.zeros(H, device=DEV), R.lengths_to_cu([100, 300, 100]).to(DEV)
    def step():
        o, stat, rest = A.packed_attention(q, k, v, cu, sink, return_stat=True)
        return (o, *A.packed_attention_backward(q, k, v, o, d_o, stat, rest, cu, sink))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for lens, seed in (([499, 1], 7), ([0, 20], 8)):
        cu.copy_(R.lengths_to_cu(lens + [0] * (3 - len(lens))).to(DEV))
        for t, s in ((q, 0), (k, 1), (v, 2), (d_o, 3)):
            t.copy_(normal(*t.shape, seed=seed * 10 + s))
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want)


def test_cut_items_repeat_bit_for_bit():
    lens = [5000, 130, 2900, 17]
    T = sum(lens)
    q, k, v, cu = normal(T, 4, 64), normal(T, 2, 64, seed=1), normal(T, 2, 64, seed=2), R.lengths_to_cu(lens).to(DEV)
    first = A.packed_attention(q, k, v, cu)
    for _ in range(20):
        assert torch.equal(A.packed_attention(q, k, v, cu), first)


def test_second_derivatives_are_refused():
    q, k = normal(20, 2, 64).requires_grad_(), normal(20, 1, 64, seed=1).requires_grad_()
    o = G.packed_attention(q, k, k, R.lengths_to_cu([20]).to(DEV))
    (dq,) = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.float().sum(), q)


def test_output_elsewhere_and_scales_out_of_range_are_refused():
    q, k, cu = normal(6, 4, 64), normal(6, 2, 64, seed=1), R.lengths_to_cu([6]).to(DEV)
    kp, vp, table = pages_of([6], 2, 64, 16)
    kv, cos = torch.tensor([6], dtype=torch.int32, device=DEV), torch.ones((16, 32), device=DEV)
    host = torch.empty(q.shape, dtype=q.dtype)
    for call in (lambda **kw: A.packed_attention(q, k, k, cu, **kw), lambda **kw: A.paged_attention(q, kp, vp, table, kv, cu, **kw),
                 lambda **kw: A.paged_append(q, k, k, kp, vp, table, kv, cos, cos, cu, **kw)):
        with pytest.raises(ValueError):
            call(out=host)
    for c in (1e300, 1e13, 1e-13, 1e-300, -1.0, float("nan")):
        with pytest.raises(ValueError):
            A.packed_attention(q, k, k, cu, c=c)
        with pytest.raises(ValueError):
            A.paged_attention(q, kp, vp, table, kv, cu, c=c)
