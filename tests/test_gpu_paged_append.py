"""New tokens into a paged cache against the formulas in 64 bits, and a run of the cache's operators together."""

import pytest
import torch

import algebraic_transformer_b200 as A
import ragged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(new, lens, H, Hkv, D, page, seed=0, start=0, tail=0, table_dtype=torch.float32, spare=3):
    g = torch.Generator().manual_seed(seed)
    T = start + sum(new) + tail
    qkv = 1.7 * torch.randn((T, (H + 2 * Hkv) * D), generator=g)
    qkv = qkv.bfloat16().to(DEV)
    used = [-(-max(n, 0) // page) for n in lens]
    width, pool = max(used + [1]) + 1, sum(used) + spare
    order = torch.randperm(pool, generator=g)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for s, u in enumerate(used):
        table[s, :u] = order[at:at + u]
        at += u
    w = 0.5 * 10000.0 ** (-torch.arange(D // 2) / (D // 2))
    cos, sin = (t.to(table_dtype).to(DEV) for t in A.cayley_powers(w, width * page))
    pages = [torch.randn((pool, page, Hkv, D), generator=g).bfloat16().to(DEV) for _ in range(2)]
    return dict(q=qkv[:, : H * D].view(T, H, D), k=qkv[:, H * D: (H + Hkv) * D].view(T, Hkv, D), v=qkv[:, (H + Hkv) * D:].view(T, Hkv, D),
                k_pages=pages[0], v_pages=pages[1], block_table=table.to(DEV), kv_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                cos=cos, sin=sin, cu_seqlens=R.lengths_to_cu(new, start).to(DEV),
                q_gain=(1 + 0.2 * torch.randn(D, generator=g)).to(DEV), k_gain=(1 + 0.2 * torch.randn(D, generator=g)).to(DEV))


def turned(x, gain, cos, sin, eps):
    """(normalised and rotated row, the sizes that were added up)"""
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    y = y if gain is None else y * gain
    a, b = y.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1), torch.cat([(a * cos).abs() + (b * sin).abs()] * 2, -1) \
        + torch.cat([(a * sin).abs() + (b * cos).abs()] * 2, -1)


def check(a, eps=1e-5, single=False):
    before = [a["k_pages"].clone(), a["v_pages"].clone()]
    call = {k: v.clone() if k.endswith("pages") else v for k, v in a.items()}
    if single:
        call["cu_seqlens"] = None
    q = A.paged_append(**call, eps=eps)
    c = {k: None if v is None else v.cpu().double() if v.is_floating_point() else v.cpu() for k, v in a.items()}
    want_k, want_v = before[0].cpu().double(), before[1].cpu().double()
    slack_k = torch.zeros_like(want_k)
    want_q, slack_q = torch.zeros_like(c["q"]), torch.zeros_like(c["q"])
    pool, page = want_k.shape[:2]
    for s, length in enumerate(c["kv_lens"].tolist()):
        lo, hi = int(c["cu_seqlens"][s]), int(c["cu_seqlens"][s + 1])
        for t in range(lo, hi):
            pos = length - (hi - lo) + t - lo
            if pos < 0:
                continue
            cs, sn = c["cos"][pos], c["sin"][pos]
            want_q[t], slack_q[t] = turned(c["q"][t], c["q_gain"], cs, sn, eps)
            number = int(c["block_table"][s, pos // page])
            if 0 <= number < pool:
                want_k[number, pos % page], slack_k[number, pos % page] = turned(c["k"][t], c["k_gain"], cs, sn, eps)
                want_v[number, pos % page] = c["v"][t]
    assert torch.equal(call["v_pages"].cpu().double(), want_v)
    # one rounding to bf16, and some twenty operations in 32 bits on what is added up
    for got, want, slack in ((q, want_q, slack_q), (call["k_pages"], want_k, slack_k)):
        off = (got.cpu().double() - want).abs()
        assert bool((off <= R.BF16 * (want.abs() + 2.0 ** -19 * slack) + 2.0 ** -19 * slack).all())
    return q


@pytest.mark.parametrize("new,lens", [([1], [1]), ([5, 0, 30], [5, 9, 130]), ([200], [256]), ([1] * 70, list(range(1, 71))), ([3, 4], [2, 0])],
                         ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("H,Hkv,D,page", [(2, 2, 64, 16), (6, 2, 64, 32), (5, 1, 128, 64), (16, 16, 128, 16), (24, 3, 64, 256)])
def test_lengths_and_heads(new, lens, H, Hkv, D, page):
    check(make(new, lens, H, Hkv, D, page, seed=len(new) + H))


@pytest.mark.parametrize("D", [64, 128])
def test_options(D):
    a = make([1] * 40, [3 * i + 1 for i in range(40)], 6, 2, D, 16, seed=2)
    check(a, single=True)
    check(dict(a, q_gain=None, k_gain=None), eps=0.5, single=True)
    b = make([9, 100], [300, 100], 4, 4, D, 32, seed=3, table_dtype=torch.bfloat16, start=3, tail=60)
    q = check(b)
    assert (q[:3] == 0).all() and (q[112:] == 0).all()
    kept = torch.full_like(b["q"], 3.0)
    A.paged_append(**dict(b, out=kept))
    assert (kept[:3] == 3).all() and (kept[112:] == 3).all() and torch.equal(kept[3:112], q[3:112])
    inplace = b["q"].clone()
    assert torch.equal(A.paged_append(**dict(b, q=inplace, out=inplace))[3:112], q[3:112])


def test_page_layouts_and_numbers_outside_the_pool():
    a = make([20, 7], [20, 90], 4, 2, 64, 32, seed=4)
    ahead = {n: a[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("k_pages", "v_pages")}
    q = A.paged_append(**dict(a, **ahead))
    plain = {n: a[n].clone() for n in ("k_pages", "v_pages")}
    assert torch.equal(q, A.paged_append(**dict(a, **plain)))
    assert all(torch.equal(ahead[n], plain[n]) for n in plain)
    a["block_table"][0, 0], a["block_table"][1, 2] = a["k_pages"].shape[0], -2 ** 31
    check(a)


def test_many_sequences_of_all_lengths():
    """The search for a token's sequence, over more than 32 x 32 of them, empty ones among them."""
    g = torch.Generator().manual_seed(5)
    new = torch.randint(0, 3, (1500,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 20, (1500,), generator=g))]
    check(make(new, lens, 1, 1, 64, 16, seed=6))


def test_prompt_in_pieces_then_single_tokens_equals_the_whole():
    """A sequence fed in chunks of different sizes and then token by token, through the cache, against its attention at one go."""
    H, Hkv, D, page, total = 6, 2, 64, 16, 150
    whole = make([total, 90], [total, 90], H, Hkv, D, page, seed=7)
    sink = 0.5 * torch.randn(H, generator=torch.Generator().manual_seed(8)).to(DEV)
    link = dict(n=16, c=8.0)
    q = A.paged_append(**whole)
    want = A.paged_attention(q, whole["k_pages"], whole["v_pages"], whole["block_table"], whole["kv_lens"], whole["cu_seqlens"], sink, **link)
    # the same prompt straight from packed keys
    keys = torch.cat([whole["k_pages"][whole["block_table"][s, : -(-n // page)].long()].reshape(-1, Hkv, D)[:n] for s, n in enumerate((total, 90))])
    packed = A.packed_attention(q, keys, whole["v"], whole["cu_seqlens"], sink, **link)
    scale = float(whole["v"].abs().max())
    assert float((packed.double() - want.double()).abs().max()) <= 4 * R.BF16 * scale
    cache = {n: torch.zeros_like(whole[n]) for n in ("k_pages", "v_pages")}
    done, got = [0, 0], torch.zeros_like(want)
    plan = [(60, 17), (1, 40), (70, 0)] + [(1, 1)] * 19 + [(0, 14)]
    for a, b in plan:
        rows = list(range(done[0], done[0] + a)) + list(range(total + done[1], total + done[1] + b))
        done = [done[0] + a, done[1] + b]
        at = torch.tensor(rows, device=DEV)
        lens = torch.tensor(done, dtype=torch.int32, device=DEV)
        cu = None if (a, b) == (1, 1) else R.lengths_to_cu([a, b]).to(DEV)
        step = dict(whole, **cache, q=whole["q"][at], k=whole["k"][at], v=whole["v"][at], kv_lens=lens, cu_seqlens=cu)
        q = A.paged_append(**step)
        got[at] = A.paged_attention(q, cache["k_pages"], cache["v_pages"], whole["block_table"], lens, cu, sink, **link)
    assert done == [total, 90]
    assert float((got.double() - want.double()).abs().max()) <= 4 * R.BF16 * scale
    used = (whole["block_table"] >= 0)
    assert torch.equal(cache["k_pages"][whole["block_table"][0, :9].long()], whole["k_pages"][whole["block_table"][0, :9].long()])
    assert used.any()
