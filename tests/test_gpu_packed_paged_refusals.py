"""Calls of the packed and paged operators that are refused, by the Python surface, ahead of any launch."""

import pytest
import torch

import algebraic_transformer_b200 as A
from algebraic_transformer_b200 import autograd as G

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def tensors():
    q = torch.zeros((6, 4, 64), dtype=torch.bfloat16, device=DEV)
    k = torch.zeros((6, 2, 64), dtype=torch.bfloat16, device=DEV)
    pages = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16, device=DEV)
    return dict(q=q, k=k, pages=pages, cu=torch.tensor([0, 6], dtype=torch.int32, device=DEV), table=torch.zeros((1, 2), dtype=torch.int32, device=DEV),
                lens=torch.tensor([6], dtype=torch.int32, device=DEV), cos=torch.ones((32, 32), device=DEV))


def test_packed_attention():
    t = tensors()
    q, k, cu = t["q"], t["k"], t["cu"]
    for bad in (dict(q=q.float()), dict(k=k[:5]), dict(v=k[:, :1]), dict(q=q[:, :3]), dict(q=q[..., :32], k=k[..., :32], v=k[..., :32]),
                dict(cu=cu.long()), dict(cu=cu[:0]), dict(cu=cu[None]), dict(sink=torch.zeros(3, device=DEV)), dict(n=12), dict(n=64), dict(c=0.0),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(q=torch.zeros((6, 1, 64), dtype=torch.bfloat16, device=DEV).expand(6, 4, 64)),
                dict(out=q.float()), dict(out=q[:5])):
        a = dict(q=q, k=k, v=k, cu=cu, sink=None, n=16, c=8.0, out=None) | bad
        with pytest.raises(ValueError):
            A.packed_attention(a["q"], a["k"], a["v"], a["cu"], a["sink"], n=a["n"], c=a["c"], out=a["out"])
    with pytest.raises(ValueError):
        G.packed_attention(q, k, k, cu, torch.zeros(4, dtype=torch.bfloat16, device=DEV))
    o, stat, rest = A.packed_attention(q, k, k, cu, return_stat=True)
    for bad in (dict(o=o.float()), dict(d_o=o[:5]), dict(stat=stat.t()), dict(stat=stat[:3]), dict(rest=rest.transpose(0, 1).contiguous().transpose(0, 1))):
        a = dict(o=o, d_o=o, stat=stat, rest=rest) | bad
        with pytest.raises(ValueError):
            A.packed_attention_backward(q, k, k, a["o"], a["d_o"], a["stat"], a["rest"], cu)


def test_paged_attention():
    t = tensors()
    good = dict(q=t["q"], k_pages=t["pages"], v_pages=t["pages"], block_table=t["table"], kv_lens=t["lens"], cu_seqlens=t["cu"])
    A.paged_attention(**good)
    for bad in (dict(q=t["q"].float()), dict(k_pages=t["pages"][:2]), dict(k_pages=t["pages"][0], v_pages=t["pages"][0]),
                dict(block_table=t["table"].long()), dict(block_table=t["table"][0]), dict(kv_lens=t["lens"].long()),
                dict(kv_lens=torch.zeros(2, dtype=torch.int32, device=DEV)), dict(cu_seqlens=None), dict(cu_seqlens=t["cu"][:1]),
                dict(k_pages=t["pages"][:, :8], v_pages=t["pages"][:, :8]), dict(n=3), dict(c=float("nan")),
                dict(block_table=torch.zeros((1, 4), dtype=torch.int32, device=DEV)[:, ::2])):
        with pytest.raises(ValueError):
            A.paged_attention(**(good | bad))
            pytest.fail(f"accepted: {bad}")


def test_paged_append():
    t = tensors()
    good = dict(q=t["q"], k=t["k"], v=t["k"], k_pages=t["pages"], v_pages=t["pages"].clone(), block_table=t["table"], kv_lens=t["lens"], cos=t["cos"],
                sin=t["cos"], cu_seqlens=t["cu"])
    A.paged_append(**good)
    gain = torch.ones(64, device=DEV)
    for bad in (dict(k=t["k"][:, :1], v=t["k"][:, :1]), dict(v=t["k"][:5]), dict(cos=t["cos"][:31], sin=t["cos"][:31]), dict(cos=t["cos"].bfloat16()),
                dict(cos=t["cos"].double(), sin=t["cos"].double()), dict(cos=t["cos"][:, :16], sin=t["cos"][:, :16]), dict(q_gain=gain[:32]),
                dict(k_gain=gain.double()), dict(eps=0.0), dict(cu_seqlens=None), dict(q=t["q"].float())):
        with pytest.raises(ValueError):
            A.paged_append(**(good | bad))
