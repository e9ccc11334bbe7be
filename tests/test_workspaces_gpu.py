"""Scratch of calls that are captured by graphs which share a stream, and of calls beside them."""
import pytest
import torch

import hidet_b200
from hidet_b200 import ffi
from hidet_b200.runtime import workspaces

pytestmark = pytest.mark.gpu
F16 = torch.float16


def operands(tokens, hidden, inner, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=gen, device='cuda').to(F16)
    router = torch.randn(8, hidden, generator=gen, device='cuda').to(F16) * 0.05
    codes = [torch.randint(-127, 128, shape, generator=gen, device='cuda', dtype=torch.int8) for shape in ((8, 2 * inner, hidden), (8, hidden, inner))]
    scales = [torch.rand(shape, generator=gen, device='cuda').to(F16) * 1e-3 for shape in ((8, 2 * inner), (8, hidden))]
    return lambda: hidet_b200.mixture_of_experts(x, *hidet_b200.route_tokens(x, router, 2), codes[0], scales[0], codes[1], scales[1])


@pytest.mark.parametrize('warm', [False, True])
def test_graphs_that_share_a_stream(warm):
    """Captured one after the other and replayed the other way round, with calls of all sizes between: none relies on what another graph has cleared, and none's scratch is given away."""
    stream = torch.cuda.Stream()
    key = (torch.cuda.current_device(), stream.cuda_stream)
    before = workspaces.swap(torch.device('cuda', key[0]), stream.cuda_stream, None)
    calls = [operands(3, 512, 768, 1), operands(40, 512, 256, 2), operands(300, 256, 512, 3)]
    want = [call() for call in calls]
    stream.wait_stream(torch.cuda.current_stream())
    graphs, results = [], []
    try:
        for call in calls:
            if warm:
                with torch.cuda.stream(stream):
                    call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = call()
                out = out + 0 * call()  # the same scratch twice
            graphs.append(graph), results.append(out)
        if not warm:  # what a graph's scratch holds before its first replay is nobody's promise
            buffer = workspaces._buffers[key]
            buffer.fill_(255)
            torch.cuda.synchronize()
        for order in ((2, 1, 0), (0, 2, 1), (1, 1, 2, 0)):
            for i in order:
                results[i].zero_()
                graphs[i].replay()
                torch.cuda.synchronize()
                assert torch.equal(results[i], want[i])
            with torch.cuda.stream(stream):
                for call, w in zip(calls, want):
                    assert torch.equal(call(), w)
            torch.cuda.synchronize()
        assert ffi.func('b200q_check_status')() == ffi.OK
    finally:
        torch.cuda.synchronize()
        workspaces.swap(torch.device('cuda', key[0]), stream.cuda_stream, before)
