"""Scratch of graphs that are captured plainly on a stream where CudaGraph objects are made as well."""
import pytest
import torch

import hidet_b200
from hidet_b200 import ffi
from hidet_b200.runtime import workspaces
from test_workspaces_gpu import operands

pytestmark = pytest.mark.gpu


def test_plain_captures_around_a_cuda_graph_on_the_same_stream():
    """torch's streams come from a pool, so a CudaGraph may get the stream of a plain capture: it puts the scratch that the capture made aside and back, and a second plain capture, and calls
    outside, do not take it for theirs.  The graph that was captured last is replayed first."""
    stream = torch.cuda.Stream()
    before = workspaces.swap(torch.device('cuda', torch.cuda.current_device()), stream.cuda_stream, None)
    calls = [operands(3, 512, 768, 1), operands(40, 512, 256, 2), operands(5, 512, 768, 3)]
    want = [call() for call in calls]
    stream.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    try:
        graphs, results = [], []
        for i in (0, 2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = calls[i]()
            graphs.append(graph), results.append(out)
            made = workspaces._buffers[(torch.cuda.current_device(), stream.cuda_stream)]
            made.fill_(255)     # what it holds before a replay is nobody's promise
            torch.cuda.synchronize()
            if i == 0:
                others = []
                while not others or others[-1]._stream.cuda_stream != stream.cuda_stream:
                    assert len(others) < 200
                    others.append(hidet_b200.CudaGraph(lambda: [torch.zeros(1, device='cuda')], lambda inputs: [calls[1]() + 0 * inputs[0].half()]))
        with torch.cuda.stream(stream):
            outside = [call() for call in calls]
        torch.cuda.synchronize()
        for got, w in zip(outside, want):
            assert torch.equal(got, w)
        for _ in range(2):
            for graph, result, i in ((graphs[1], results[1], 2), (graphs[0], results[0], 0)):
                result.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(result, want[i])
            assert torch.equal(others[-1].run()[0], want[1])
        assert ffi.func('b200q_check_status')() == ffi.OK
    finally:
        torch.cuda.synchronize()
        workspaces.swap(torch.device('cuda', torch.cuda.current_device()), stream.cuda_stream, before)


def test_plain_captures_on_a_stream_that_is_warm_are_replayed_at_the_same_time():
    """Each has scratch of its own, also where calls outside have left some on the stream."""
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    calls = [operands(40, 1024, 768, 1), operands(33, 1024, 512, 2)]
    want = [call() for call in calls]
    graphs, results = [], []
    stream.wait_stream(torch.cuda.current_stream())
    for call in calls:
        with torch.cuda.stream(stream):
            call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            results.append(call())
        graphs.append(graph)
    torch.cuda.synchronize()
    for i in range(40):
        for s, graph, result in zip((stream, other), graphs, results):
            with torch.cuda.stream(s):
                graph.replay()
                if i % 4 == 0:
                    calls[0]()     # and calls outside beside them
        if i % 8 == 7:
            torch.cuda.synchronize()
            for result, w in zip(results, want):
                assert torch.equal(result, w)
                result.zero_()
            torch.cuda.synchronize()
    assert ffi.func('b200q_check_status')() == ffi.OK
