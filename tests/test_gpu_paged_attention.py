"""Attention over a paged cache, chunks and single tokens, against its definition in 64 bits."""

import pytest
import torch

import algebraic_transformer_b200 as A
import ragged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(new, lens, H, Hkv, D, page, seed=0, size=1.0, start=0, tail=0, garbage=True, spare=3):
    """A pool whose pages are used in no order; rows behind a sequence's end, unused pages and unused table entries hold anything."""
    g = torch.Generator().manual_seed(seed)
    T = start + sum(new) + tail
    unit = lambda t: t / t.square().mean(-1, keepdim=True).sqrt().clamp_min(1e-9)   # noqa: E731
    q = size * unit(torch.randn((T, H, D), generator=g))
    used = [-(-n // page) for n in lens]
    width, pool = max(used + [1]) + 2, sum(used) + spare
    k, v = size * unit(torch.randn((pool, page, Hkv, D), generator=g)), torch.randn((pool, page, Hkv, D), generator=g)
    order = torch.randperm(pool, generator=g)
    table = torch.full((len(lens), width), 2 ** 31 - 7 if garbage else 0, dtype=torch.int64)
    at = 0
    for s, u in enumerate(used):
        table[s, :u] = order[at:at + u]
        if garbage and u and lens[s] % page:
            k[table[s, u - 1], lens[s] % page:] = float("nan")
            v[table[s, u - 1], lens[s] % page:] = float("nan")
        at += u
    if garbage:
        k[order[at:]], v[order[at:]] = float("inf"), float("nan")
        q[:start], q[start + sum(new):] = float("nan"), float("inf")
    sink = 0.7 * torch.randn(H, generator=g)
    cu = R.lengths_to_cu(new, start).to(DEV)
    return dict(q=q.bfloat16().to(DEV), k_pages=k.bfloat16().to(DEV), v_pages=v.bfloat16().to(DEV), block_table=table.to(torch.int32).to(DEV),
                kv_lens=torch.tensor(lens, dtype=torch.int32, device=DEV), cu_seqlens=cu, sink_logit=sink.to(DEV))


def check(a, n=16, c=8.0, single=False):
    a = dict(a)
    if single:
        a["cu_seqlens"] = None
    o = A.paged_attention(**a, n=n, c=c)
    ref, spread, err = R.paged(a["q"], a["k_pages"], a["v_pages"], a["block_table"], a["kv_lens"].tolist(), a["cu_seqlens"],
                               a["sink_logit"], n, c)
    R.assert_close(o, ref, spread, err)
    return o


CHUNKS = [([1], [1]), ([5, 1, 30], [5, 100, 30]), ([128, 0, 129], [400, 77, 129]), ([0, 0], [10, 0]), ([3, 200], [255, 256]), ([17], [1030])]


@pytest.mark.parametrize("new,lens", CHUNKS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("H,Hkv,D,page", [(2, 2, 64, 16), (6, 2, 64, 32), (4, 1, 128, 64), (16, 2, 128, 128), (3, 1, 64, 256), (2, 1, 128, 16)])
def test_chunks(new, lens, H, Hkv, D, page):
    check(make(new, lens, H, Hkv, D, page, seed=len(lens) + page))


@pytest.mark.parametrize("lens", [[1], [31, 32, 33, 64, 65], [0, 5, 0], [1000, 1, 400], [2500]], ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("H,Hkv,D,page", [(2, 2, 64, 16), (6, 2, 64, 32), (8, 1, 128, 64), (12, 1, 128, 16), (16, 1, 64, 128), (40, 2, 64, 16),
                                          (34, 1, 128, 256)])
def test_single_tokens(lens, H, Hkv, D, page):
    a = make([1] * len(lens), lens, H, Hkv, D, page, seed=len(lens) + H)
    one = check(a, single=True)
    chunk = A.paged_attention(**a)
    assert float((one.double() - chunk.double()).abs().max()) <= 4 * R.BF16 * float(a["v_pages"][a["v_pages"].isfinite()].abs().max())


@pytest.mark.parametrize("n", [2, 4, 8, 16, 32])
@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("size", [0.05, 1.0, 6.0])
def test_powers_and_score_sizes(n, single, size):
    new = [1, 1, 1] if single else [40, 1, 9]
    for D in (64, 128):
        a = make(new, [200, 61, 9], 3, 1, D, 32, seed=n, size=size)
        check(a, n=n, c=8.0 if size < 2 else 3.0, single=single)
        a["sink_logit"] = None
        check(a, n=n, c=8.0 if size < 2 else 3.0, single=single)


@pytest.mark.parametrize("single", [False, True])
def test_long_caches_are_cut_along_the_keys(single):
    new = [1, 1] if single else [3, 50]
    for H, Hkv, D in ((4, 1, 64), (2, 2, 128), (16, 1, 128)):
        a = make(new, [5000, 2100], H, Hkv, D, 64, seed=H)
        check(a, single=single)
        a["q"] *= 60
        check(a, single=single)


@pytest.mark.parametrize("single", [False, True])
def test_fewer_keys_than_new_tokens(single):
    """Tokens ahead of the sequence's first key see nothing: zero, with a sink or without."""
    a = make([1, 1] if single else [7, 40], [0, 30], 4, 2, 64, 16, seed=3)
    o = check(a, single=single)
    a["sink_logit"] = None
    assert torch.isfinite(check(a, single=single).float()).all()
    if not single:
        assert (o[:7] == 0).all() and (o[7:17] == 0).all() and (o[17] != 0).any()


def test_rows_of_no_sequence_and_out():
    a = make([9, 0, 20], [30, 12, 300], 4, 2, 128, 32, seed=4, start=5, tail=33)
    o = check(a)
    assert (o[:5] == 0).all() and (o[34:] == 0).all()
    kept = torch.full_like(a["q"], 3.0)
    A.paged_attention(**a, out=kept)
    assert (kept[:5] == 3).all() and (kept[34:] == 3).all() and torch.equal(kept[5:34], o[5:34])


@pytest.mark.parametrize("single", [False, True])
def test_cache_layouts(single):
    """Heads ahead of the rows of a page; both caches in one pool; rows of a wider table."""
    a = make([1, 1] if single else [20, 3], [100, 230], 4, 2, 64, 32, seed=5, garbage=False)
    want = check(a, single=single)
    if single:
        a["cu_seqlens"] = None
    b = dict(a)
    for name in ("k_pages", "v_pages"):
        b[name] = a[name].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(A.paged_attention(**b), want)
    both = torch.stack([a["k_pages"], a["v_pages"]], dim=1)
    b["k_pages"], b["v_pages"] = both[:, 0], both[:, 1]
    assert torch.equal(A.paged_attention(**b), want)
    wide = torch.zeros((2, 40), dtype=torch.int32, device=DEV)
    wide[:, : a["block_table"].shape[1]] = a["block_table"]
    b["block_table"] = wide[:, : a["block_table"].shape[1]]
    assert torch.equal(A.paged_attention(**b), want)


@pytest.mark.parametrize("single", [False, True])
def test_lengths_and_pages_that_lead_outside(single):
    a = make([1, 1] if single else [20, 3], [100, 230], 4, 2, 64, 32, seed=6, garbage=False)
    if single:
        a["cu_seqlens"] = None
    width = a["block_table"].shape[1]
    a["block_table"][0, 1], a["block_table"][1, 3] = -1, a["k_pages"].shape[0]           # read as zeros
    check(a, single=single)
    most = dict(a, kv_lens=torch.tensor([2 ** 31 - 1, width * 32], dtype=torch.int32, device=DEV))
    full = dict(a, kv_lens=torch.tensor([width * 32, width * 32], dtype=torch.int32, device=DEV))
    assert torch.equal(A.paged_attention(**most), A.paged_attention(**full))
    none = dict(a, kv_lens=torch.tensor([-3, 0], dtype=torch.int32, device=DEV))
    assert (A.paged_attention(**none) == 0).all()


@pytest.mark.parametrize("single", [False, True])
def test_graph_replayed_as_the_sequences_grow(single):
    a = make([1, 1] if single else [20, 3], [100, 230], 4, 2, 64, 32, seed=7, garbage=False)
    if single:
        a["cu_seqlens"] = None
    want = [A.paged_attention(**dict(a, kv_lens=a["kv_lens"] - i)) for i in (0, 30, 60)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    held = dict(a, kv_lens=a["kv_lens"].clone())
    with torch.cuda.stream(side):
        A.paged_attention(**held)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):                                             # two graphs of one call: each has its own scratch
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(A.paged_attention(**held))
    for i, w in zip((60, 0, 30, 0), (want[2], want[0], want[1], want[0])):
        held["kv_lens"].copy_(a["kv_lens"] - i)
        for graph in graphs:
            graph.replay()
        assert torch.equal(outs[0], w) and torch.equal(outs[1], w)
