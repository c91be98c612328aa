"""Products that follow the quantiser on the same stream, on more streams than one hand counts and around a capture."""
import pytest
import torch

import vq_gemm_b200 as V
from tests.test_gpu_int4 import F16, acts
from vq_gemm_b200 import quantize

pytestmark = pytest.mark.gpu


def dense(seed, n=2048, k=2048):
    return (torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) * 0.05).half().cuda()


def test_quantised_on_forty_streams_and_multiplied_there():
    x, ws = acts(2, 2048, F16), [dense(s) for s in range(40)]
    want = [V.int4_gemm(x, *quantize.int4_quantize(w)) for w in ws]
    many = acts(64, 2048, F16)
    streams = [torch.cuda.Stream() for _ in ws]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for w, s in zip(ws, streams):          # marks left behind by products of many rows, which do not clear them
            with torch.cuda.stream(s):
                V.int4_gemm(many, *quantize.int4_quantize(w))
        for w, s in zip(ws, streams):
            with torch.cuda.stream(s):
                got.append(V.int4_gemm(x, *quantize.int4_quantize(w)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_quantised_eagerly_before_a_capture_and_inside_one():
    side, x, w = torch.cuda.Stream(), acts(2, 2048, F16), dense(1)
    q = quantize.int4_quantize(w)
    want = V.int4_gemm(x, *q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        fresh = quantize.int4_quantize(w)      # a mark of the stream itself
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            inside = V.int4_gemm(x, *fresh)
            own = V.int4_gemm(x, *quantize.int4_quantize(w))
        eager = V.int4_gemm(x, *fresh)
        for _ in range(3):
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager, want) and torch.equal(inside, want) and torch.equal(own, want)
