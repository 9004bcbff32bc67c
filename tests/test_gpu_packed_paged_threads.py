"""Calls of the packed and paged operators from several threads at once, on one stream and on streams of their own."""

import threading

import pytest
import torch

import algebraic_transformer_b200 as A
from test_gpu_packed_attention import make
from test_gpu_paged_attention import make as make_paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("own_stream", [False, True])
def test_threads(own_stream):
    q, k, v, sink, cu = make([300, 2300, 41], 4, 2, 64, seed=1)
    d_o = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    paged = make_paged([1, 40, 7], [900, 400, 2600], 4, 2, 64, 32, seed=3)
    single = dict(make_paged([1] * 5, [900, 1, 400, 33, 2600], 6, 2, 64, 16, seed=4), cu_seqlens=None)

    def train():
        o, stat, rest = A.packed_attention(q, k, v, cu, sink, return_stat=True)
        return (o, *A.packed_attention_backward(q, k, v, o, d_o, stat, rest, cu, sink))

    jobs = [train, lambda: (A.packed_attention(q, k, v, cu, sink),), lambda: (A.paged_attention(**paged),), lambda: (A.paged_attention(**single),)] * 2
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    failures, start = [], threading.Barrier(len(jobs))

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream() if own_stream else torch.cuda.current_stream()):
                start.wait()
                outs = [jobs[i]() for _ in range(20)]
                torch.cuda.current_stream().synchronize()
                for out in outs:
                    if not all(torch.equal(a, b) for a, b in zip(out, want[i])):
                        failures.append(i)
        except Exception as e:  # noqa: BLE001
            failures.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
