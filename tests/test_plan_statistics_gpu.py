"""Operators captured into a graph before anybody has asked for the statistics of their plan."""
import pytest
import torch

from torchex_b200 import ScatterData, gather_back, scatter_max, scatter_mean, scatter_sum, segment_attention

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _data():
    ids = torch.arange(500, device=DEV) * 7 % 40
    return ScatterData(ids, torch.bincount(ids, minlength=40))


@pytest.mark.parametrize("call", [
    lambda x, d: scatter_sum(x, d), lambda x, d: scatter_mean(x, d), lambda x, d: scatter_max(x, d)[0],
    lambda x, d: gather_back(scatter_sum(x, d), d),
    lambda x, d: segment_attention(*(x.half().view(500, 2, 16),) * 3, d)])
def test_capture_right_after_the_plan(call):
    x = torch.randn(500, 32, device=DEV)
    want = call(x, _data())
    data = _data()
    assert data._pending is not None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(x, data)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert data.max_cnt == 13
