"""Layers of experts straight behind one another, without another kernel or a wait between: each goes by its own tokens' experts, whatever stood in the same scratch before."""
import pytest
import torch

import hidet_b200
from hidet_b200 import ffi
from test_experts_gpu import choices, generator, layer, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('tokens,count,top,hidden,inner', [(1, 8, 2, 512, 768), (30, 8, 2, 1024, 512), (200, 8, 2, 512, 768), (600, 64, 4, 256, 512), (90, 200, 6, 256, 128), (5, 6, 2, 50, 36)])
@pytest.mark.parametrize('captured', [False, True])
def test_choices_in_turn(tokens, count, top, hidden, inner, captured):
    gen = generator(tokens, count)
    x, w = normal(gen, tokens, hidden, dtype=torch.float16), layer(gen, count, hidden, inner)
    picks = [choices(gen, tokens, count, top) for _ in range(3)]
    one = torch.full_like(picks[0][0], count // 2)     # all to one expert: another number of entries, groups and slots
    picks.append((one, picks[0][1]))
    picks.append((torch.full_like(one, -1), picks[0][1]))
    want = []
    for e, p in picks:
        want.append(hidet_b200.mixture_of_experts(x, e, p, *w))
        torch.cuda.synchronize()
    order = [0, 3, 1, 2, 4, 1, 0, 4, 3, 2] * 3

    def run():
        return [hidet_b200.mixture_of_experts(x, *picks[i], *w) for i in order]

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        graph.replay()
    else:
        got = run()
    for i, g in zip(order, got):
        assert torch.equal(g, want[i])
    assert ffi.func('b200q_check_status')() == ffi.OK
