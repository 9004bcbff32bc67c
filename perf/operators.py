"""Attention over packed sequences and over a paged cache, as cases that can be timed and compared.

Sequences of different lengths lie one behind the other in (tokens, heads, head_dim) tensors, query heads share key heads in
groups, and a cache is a pool of pages with a table of them per sequence.  Every weight is the `algebraic` preset's:
rho(x)^n of x = q.k / (sqrt(head_dim) c), with a learned sink per head in the denominator.  Heads and head sizes are those of the
model presets (6, 12, 16, 24 heads of 64) and of the benchmark's attention (16 heads of 128), whole or grouped.

A case is a dict of plain values; `kind` says which call it is:

    prompt   causal attention of packed sequences (inference)
    train    the same, forward and backward through torch.autograd: q, k, v and the sinks
    token    one new token of each sequence against its pages (generation)
    chunk    several new tokens of each sequence against its pages, which hold the chunk's own keys too (prompts in
             pieces, drafts to be verified, both beside single tokens)
    append   QK-norm, rotation by the tokens' own positions and the write of their keys and values into the pages

Lengths are spread over their range by logarithm, from `shortest` to `longest`, the longest always among them; `mix` numbers
the draw.  `new` is the longest chunk (1: every sequence has one new token).
"""

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
N, C, EPS = 16, 8.0, 1e-5       # the `algebraic` preset's attention link and the norms' epsilon


def listed():
    return [
        # three short questions that arrive together at the 125M model: all latency
        dict(name="prompt_few", kind="prompt", heads=12, kv_heads=4, head_dim=64, sequences=3, shortest=5, longest=90, mix=1),
        # a prefill batch of the 350M model, prompts of all lengths
        dict(name="prompt_mixed", kind="prompt", heads=16, kv_heads=4, head_dim=64, sequences=24, shortest=17, longest=2001, mix=2),
        # two documents with the heads of the long-sequence benchmark, eight queries to a key head
        dict(name="prompt_long", kind="prompt", heads=16, kv_heads=2, head_dim=128, sequences=2, shortest=5000, longest=8192, mix=3),
        # a training batch of the 125M model's heads, documents packed up to its length
        dict(name="train_mixed", kind="train", heads=12, kv_heads=4, head_dim=64, sequences=20, shortest=60, longest=1024, mix=4),
        # longer documents at head size 128, every query head with a key head of its own
        dict(name="train_long", kind="train", heads=16, kv_heads=16, head_dim=128, sequences=3, shortest=901, longest=4096, mix=5),
        # the first tokens of one generation: the smallest call there is
        dict(name="token_first", kind="token", heads=12, kv_heads=12, head_dim=64, sequences=1, shortest=333, longest=333, new=1,
             page=16, mix=6),
        # a serving batch of the 1B model
        dict(name="token_batch", kind="token", heads=24, kv_heads=8, head_dim=64, sequences=64, shortest=70, longest=4001, new=1,
             page=64, mix=7),
        # a few long contexts
        dict(name="token_long", kind="token", heads=16, kv_heads=2, head_dim=128, sequences=4, shortest=20000, longest=60001, new=1,
             page=128, mix=8),
        # continuous batching: pieces of prompts beside drafts and single tokens
        dict(name="chunk_mixed", kind="chunk", heads=16, kv_heads=4, head_dim=64, sequences=32, shortest=40, longest=4000, new=512,
             page=16, mix=9),
        # two long prompts in pieces of up to 2048
        dict(name="chunk_long", kind="chunk", heads=16, kv_heads=4, head_dim=128, sequences=2, shortest=20000, longest=30001, new=2048,
             page=64, mix=34),
        # the new tokens of a generating batch
        dict(name="append_tokens", kind="append", heads=24, kv_heads=8, head_dim=64, sequences=64, shortest=70, longest=4001, new=1,
             page=64, mix=11),
        # a prefill batch's tokens
        dict(name="append_prompts", kind="append", heads=16, kv_heads=16, head_dim=128, sequences=24, shortest=300, longest=2001,
             new=2001, page=32, mix=12),
    ]


HEADS = [(6, 6, 64), (6, 2, 64), (12, 12, 64), (12, 4, 64), (16, 4, 64), (16, 16, 64), (24, 8, 64), (24, 3, 64), (16, 2, 128), (16, 4, 128),
         (16, 16, 128), (12, 2, 128)]


def draw(rng):
    while True:
        kind = rng.choice(["prompt", "train", "token", "chunk", "append"])
        heads, kv_heads, head_dim = rng.choice(HEADS)
        case = dict(kind=kind, heads=heads, kv_heads=kv_heads, head_dim=head_dim, mix=rng.randrange(1 << 20))

        def spread(low, high):
            return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

        top = {"prompt": 8192, "train": 4096, "token": 60000, "chunk": 30000, "append": 8000}[kind]
        case["longest"] = spread(20, top)
        case["shortest"] = spread(1, case["longest"])
        case["sequences"] = spread(1, 64)
        if kind in ("token", "chunk", "append"):
            case["page"] = rng.choice([16, 32, 64, 128, 256])
            case["new"] = 1 if kind == "token" else spread(1, min(case["longest"], 2048))
        # no more scores (padded to the longest) and no more bytes than the listed cases'
        queries = case["longest"] if kind in ("prompt", "train") else case["new"]
        scores = case["sequences"] * heads * queries * case["longest"]
        most = {"prompt": 2 * 16 * 8192 * 8192, "train": 3 * 16 * 4096 * 4096}.get(kind, 2 * 16 * 2048 * 30001)
        if scores <= most and work(case)["bytes"] <= 1.6e8 and case["sequences"] * case["longest"] <= 250000:
            return case


# ------------------------------------------------------------------------------------ lengths and inputs

def lengths(case):
    """(new tokens, all keys) of each sequence, as lists: plain functions of the case."""
    rng = random.Random(case["mix"])
    low, high = math.log(case["shortest"]), math.log(case["longest"])
    keys = [case["longest"]] + [int(round(math.exp(rng.uniform(low, high)))) for _ in range(case["sequences"] - 1)]
    rng.shuffle(keys)
    if case["kind"] in ("prompt", "train"):
        return list(keys), keys
    if case["new"] == 1:
        return [1] * len(keys), keys
    new = [min(k, int(round(math.exp(rng.uniform(0.0, math.log(case["new"])))))) for k in keys]
    most = keys.index(max(keys))
    new[most] = min(keys[most], case["new"])
    return new, keys


def pairs(case):
    """How many (token, key) pairs are visible, over the sequences."""
    new, keys = lengths(case)
    return sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(new, keys))


def work(case):
    new, keys = lengths(case)
    H, Hkv, D, T = case["heads"], case["kv_heads"], case["head_dim"], sum(new)
    product = 4.0 * D * H * pairs(case)                           # scores and weighted values
    if case["kind"] == "prompt":
        return {"bytes": 2.0 * T * D * (2 * H + 2 * Hkv), "flops": product}
    if case["kind"] == "train":                                   # q, dO, o, dq and k, v, dk, dv
        return {"bytes": 2.0 * T * D * (4 * H + 4 * Hkv) + 8.0 * H, "flops": 3.5 * product}
    if case["kind"] == "append":                                  # q, k, v in and out, a row of cosines and sines a token
        return {"bytes": 2.0 * T * D * (2 * H + 4 * Hkv) + 4.0 * T * D, "flops": 10.0 * T * D * (H + Hkv)}
    return {"bytes": 2.0 * D * (2 * H * T + 2 * Hkv * sum(keys)) + 4.0 * sum(-(-k // case["page"]) for k in keys), "flops": product}


def _unit_rows(t):
    return t / torch.sqrt(torch.mean(t * t, dim=-1, keepdim=True) + EPS)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    new, keys = lengths(case)
    T, S = sum(new), len(new)
    s = dict(kind=case["kind"], longest=max(keys), longest_new=max(new))
    s["sink"] = 0.5 * normal(H)
    s["cu_seqlens"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(DEVICE)
    if case["kind"] == "append":                                  # as a projection leaves them: q | k | v beside each other
        qkv = (1.5 * normal(T, (H + 2 * Hkv) * D)).bfloat16()
        s["q"] = qkv[:, : H * D].view(T, H, D)
        s["k"] = qkv[:, H * D: (H + Hkv) * D].view(T, Hkv, D)
        s["v"] = qkv[:, (H + Hkv) * D:].view(T, Hkv, D)
        s["q_gain"], s["k_gain"] = 1.0 + 0.1 * normal(D), 1.0 + 0.1 * normal(D)
    else:                                                         # q and k come normalised, as the models have them
        s["q"] = _unit_rows(normal(T, H, D)).bfloat16()
    if case["kind"] in ("prompt", "train"):
        s["k"] = _unit_rows(normal(T, Hkv, D)).bfloat16()
        s["v"] = normal(T, Hkv, D).bfloat16()
        if case["kind"] == "train":
            s["d_o"] = normal(T, H, D).bfloat16()
            s["leaves"] = [s[name].clone().requires_grad_() for name in ("q", "k", "v", "sink")]
        return s
    # the pool holds a quarter more pages than are in use; the sequences' pages lie in it in no order
    page = case["page"]
    used = [-(-k // page) for k in keys]
    width, pool = max(used), sum(used) + sum(used) // 4 + 1
    order = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
    table = np.full((S, width), 0, dtype=np.int64)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = np.arange(at, at + u)
        at += u
    s["block_table"] = order[torch.from_numpy(table).to(DEVICE)].contiguous()
    s["kv_lens"] = torch.tensor(keys, dtype=torch.int32, device=DEVICE)
    s["k_pages"] = _unit_rows(normal(pool, page, Hkv, D)).bfloat16()
    s["v_pages"] = normal(pool, page, Hkv, D).bfloat16()
    if case["new"] == 1:
        s["cu_seqlens"] = None                                    # one token a sequence
    if case["kind"] == "append":                                  # the Cayley rotation's tables over the cache's whole length
        step = 2.0 * np.arctan(0.5 * 10000.0 ** (-np.arange(D // 2) / (D // 2)))
        angle = np.arange(width * page)[:, None] * step[None, :]
        s["cos"] = torch.from_numpy(np.cos(angle).astype(np.float32)).to(DEVICE)
        s["sin"] = torch.from_numpy(np.sin(angle).astype(np.float32)).to(DEVICE)
    return s


# ------------------------------------------------------------------------------------ plain forms

def _cu(s):
    rows = s["q"].shape[0]
    return torch.arange(rows + 1, device=s["q"].device) if s["cu_seqlens"] is None else s["cu_seqlens"].long()


def _places(s):
    """(sequence, place among its sequence's new tokens) of each token."""
    cu = _cu(s)
    token = torch.arange(s["q"].shape[0], device=cu.device)
    sequence = torch.searchsorted(cu, token, right=True) - 1
    return sequence, token - cu[sequence]


def _padded(packed, s, sequence, place, length):
    """(T, heads, D) -> (S, heads, length, D) in 32 bits, zeros behind each sequence."""
    out = torch.zeros((_cu(s).numel() - 1, length) + packed.shape[1:], device=packed.device)
    out[sequence, place] = packed.float()
    return out.transpose(1, 2)


def _weights(q, k, visible, sink):
    """x (S,Hkv,G,Lq,Lk) and the normalised weights; the sink's normalised weight (S,Hkv,G,Lq,1)."""
    S, H, Lq, D = q.shape
    Hkv = k.shape[1]
    x = torch.matmul(q.reshape(S, Hkv, -1, D), k.transpose(-1, -2)).view(S, Hkv, H // Hkv, Lq, -1).mul_(1.0 / (math.sqrt(D) * C))
    b = (N * torch.asinh(sink / C)).view(1, Hkv, H // Hkv, 1, 1)
    a = torch.asinh(x).mul_(N).masked_fill_(~visible[:, None, None], -math.inf)
    top = torch.maximum(a.amax(dim=-1, keepdim=True), b)
    w = a.sub_(top).exp_()
    of_sink = torch.exp(b - top)
    total = w.sum(dim=-1, keepdim=True) + of_sink
    return x, w.div_(total), of_sink / total


def _plain_packed(s):
    sequence, place = _places(s)
    q, k, v = (_padded(s[name], s, sequence, place, s["longest"]) for name in ("q", "k", "v"))
    at = torch.arange(s["longest"], device=q.device)
    length = (_cu(s)[1:] - _cu(s)[:-1])[:, None, None]
    visible = (at[None, :, None] >= at[None, None, :]) & (at[None, None, :] < length)
    S, H, L, D = q.shape
    Hkv = k.shape[1]
    x, p, p_sink = _weights(q, k, visible, s["sink"])
    o = torch.matmul(p.view(S, Hkv, -1, L), v)                                   # (S, Hkv, G L, D)

    def packed(t):
        return t.reshape(S, -1, L, D).transpose(1, 2)[sequence, place].bfloat16()

    if s["kind"] == "prompt":
        return packed(o)
    d_o = _padded(s["d_o"], s, sequence, place, L).reshape(S, Hkv, -1, D)
    delta = (d_o * o).sum(dim=-1).view(S, Hkv, H // Hkv, L, 1)
    dv = torch.matmul(p.view(S, Hkv, -1, L).transpose(-1, -2), d_o)
    slope = x.square_().add_(1.0).rsqrt_()
    ds = torch.matmul(d_o, v.transpose(-1, -2)).view_as(p).sub_(delta).mul_(p).mul_(slope).mul_(N / (math.sqrt(D) * C)).view(S, Hkv, -1, L)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q.reshape(S, Hkv, -1, D))
    dsink = -(N / C) * torch.rsqrt(1.0 + (s["sink"] / C).square()) * (p_sink * delta).double().sum(dim=(0, 3, 4)).reshape(H).float()
    return [packed(o), packed(dq), packed(dk), packed(dv), dsink]


def _plain_paged(s):
    sequence, place = _places(s)
    q = _padded(s["q"], s, sequence, place, s["longest_new"])
    S, H, Lq, D = q.shape
    lens = s["kv_lens"].long()
    Lk = s["longest"]
    key = torch.arange(Lk, device=q.device)
    page = s["k_pages"].shape[1]
    at = s["block_table"].long()[:, key // page]                                 # (S, Lk)
    there = key[None] < lens[:, None]
    k, v = ((s[name][at, key % page].float() * there[:, :, None, None]).transpose(1, 2) for name in ("k_pages", "v_pages"))
    first = lens - (_cu(s)[1:] - _cu(s)[:-1])                                    # the first new token's position
    position = first[:, None] + torch.arange(Lq, device=q.device)[None]
    visible = (key[None, None] <= position[:, :, None]) & there[:, None]
    _, p, _ = _weights(q, k, visible, s["sink"])
    o = torch.matmul(p.view(S, k.shape[1], -1, Lk), v).reshape(S, H, Lq, D)
    return o.transpose(1, 2)[sequence, place].bfloat16()


def _plain_append(s):
    sequence, place = _places(s)
    position = (s["kv_lens"].long() - (_cu(s)[1:] - _cu(s)[:-1]))[sequence] + place
    page = s["k_pages"].shape[1]
    where = (s["block_table"].long()[sequence, position // page], position % page)
    cos, sin = s["cos"][position][:, None], s["sin"][position][:, None]

    def rotated(x, gain):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + EPS) * gain
        a, b = y.chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1).bfloat16()

    s["k_pages"][where] = rotated(s["k"], s["k_gain"])
    s["v_pages"][where] = s["v"]
    return [rotated(s["q"], s["q_gain"]), s["k_pages"], s["v_pages"]]


def run(state):
    s = state
    if own:
        import algebraic_transformer_b200 as A
        from algebraic_transformer_b200 import autograd as G

        if s["kind"] == "prompt":
            return A.packed_attention(s["q"], s["k"], s["v"], s["cu_seqlens"], s["sink"], n=N, c=C)
        if s["kind"] == "train":
            q, k, v, sink = s["leaves"]
            o = G.packed_attention(q, k, v, s["cu_seqlens"], sink, n=N, c=C)
            return [o.detach(), *torch.autograd.grad(o, s["leaves"], s["d_o"])]
        if s["kind"] == "append":
            q = A.paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["block_table"], s["kv_lens"], s["cos"], s["sin"],
                               s["cu_seqlens"], q_gain=s["q_gain"], k_gain=s["k_gain"], eps=EPS)
            return [q, s["k_pages"], s["v_pages"]]
        return A.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["kv_lens"], s["cu_seqlens"], s["sink"], n=N, c=C)
    if s["kind"] == "append":
        return _plain_append(s)
    if s["kind"] in ("prompt", "train"):
        return _plain_packed(s)
    return _plain_paged(s)


# ------------------------------------------------------------------------------------ the definition in 64 bits

def _defined(q, k, v, sink, first):
    """Attention of one sequence's heads, q (H, Lq, D) over k, v (Hkv, Lk, D); token i stands at position first + i."""
    H, Lq, D = q.shape
    k, v = (t.repeat_interleave(H // t.shape[0], dim=0) for t in (k, v))
    x = (q @ k.transpose(1, 2)) / (D ** 0.5 * C)
    root = torch.sqrt(1.0 + x * x)
    rho = torch.where(x >= 0, x + root, 1.0 / (root - x))
    hidden = torch.arange(k.shape[1], device=q.device)[None] > first + torch.arange(Lq, device=q.device)[:, None]
    w = rho.pow(N).masked_fill(hidden, 0.0)
    z = sink / C
    return (w @ v) / (w.sum(-1, keepdim=True) + (z + torch.sqrt(1.0 + z * z)).pow(N)[:, None, None])


def exact(case, seed):
    s = prepare(case, seed)
    new, keys = lengths(case)
    starts = np.concatenate([[0], np.cumsum(new)])
    Hkv, G = case["kv_heads"], case["heads"] // case["kv_heads"]
    if case["kind"] in ("prompt", "train"):
        train = case["kind"] == "train"
        out = [torch.zeros(s[n].shape, dtype=torch.float64, device=DEVICE) for n in (("q", "q", "k", "v", "sink") if train else ("q",))]
        for i, length in enumerate(new):
            rows = slice(int(starts[i]), int(starts[i]) + length)
            for h in range(Hkv):                                  # a key head at a time: little memory
                group = slice(h * G, (h + 1) * G)
                q, k, v = s["q"][rows, group].double(), s["k"][rows, h:h + 1].double(), s["v"][rows, h:h + 1].double()
                q, k, v, b = (t.requires_grad_(train) for t in (q, k, v, s["sink"][group].double()))
                o = _defined(q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1), b, 0).transpose(0, 1)
                out[0][rows, group] = o.detach()
                if train:
                    gq, gk, gv, gb = torch.autograd.grad(o, (q, k, v, b), s["d_o"][rows, group].double())
                    out[1][rows, group], out[2][rows, h:h + 1], out[3][rows, h:h + 1] = gq, gk, gv
                    out[4][group] += gb
        return out if train else out[0]
    page = case["page"]
    if case["kind"] == "append":
        q = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        half = case["head_dim"] // 2
        for i, length in enumerate(new):
            rows = slice(int(starts[i]), int(starts[i]) + length)
            position = torch.arange(keys[i] - length, keys[i], device=DEVICE)
            turn = torch.complex(s["cos"][position].double(), s["sin"][position].double())[:, None]
            slot = s["block_table"][i, position // page].long() * page + position % page
            for name, gain, to in (("q", "q_gain", None), ("k", "k_gain", k_pages)):
                y = s[name][rows].double()
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / (2 * half) + EPS) * s[gain].double()
                z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
                y = torch.cat([z.real, z.imag], dim=-1)
                if to is None:
                    q[rows] = y
                else:
                    to.view(-1, *to.shape[2:])[slot] = y
            v_pages.view(-1, *v_pages.shape[2:])[slot] = s["v"][rows].double()
        return [q, k_pages, v_pages]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for i, length in enumerate(new):
        rows = slice(int(starts[i]), int(starts[i]) + length)
        used = s["block_table"][i, : -(-keys[i] // page)].long()
        for h in range(Hkv):
            k, v = (s[name][used][:, :, h].reshape(-1, case["head_dim"])[: keys[i]].double()[None] for name in ("k_pages", "v_pages"))
            group = slice(h * G, (h + 1) * G)
            out[rows, group] = _defined(s["q"][rows, group].double().transpose(0, 1), k, v, s["sink"][group].double(),
                                        keys[i] - length).transpose(0, 1)
    return out
