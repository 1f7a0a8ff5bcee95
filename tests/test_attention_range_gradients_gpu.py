"""Gradients of the attention within segments on fp16 values whose gradients of scores, or probabilities, are far below
fp16's smallest normal number (bounds: test_attention_range_gpu)."""
import pytest
import torch

from tests.test_attention_gpu import DEV, _inputs, _plan, _step
from tests.test_attention_range_gpu import H, SHAPES, STEP, _check, _definition, _peaked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,dim", SHAPES)
@pytest.mark.parametrize("below", [18, 26])
def test_small_probabilities_reach_the_gradients(lens, dim, below):
    ids, data = _plan(lens, False)
    parts = [_peaked(n, 2, dim, below) for n in lens]
    q, k, v, g = (torch.cat(x) for x in zip(*parts))
    _check(_step(q, k, v, g, data, scale=1.0)[1:], _definition(q, k, v, g, lens, False, 1.0)[1:], ("g_q", "g_k", "g_v"))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,dim", [([700], 16), ([40, 64, 3], 32), ([2048], 64), ([2300, 1, 300], 128)])
@pytest.mark.parametrize("power", [-10, -14, 4])
def test_gradients_of_any_size(lens, dim, causal, power):
    ids, data = _plan(lens, False)
    q, k, v, g = _inputs(sum(lens), 2, 2, dim, torch.float16, dim)
    g = (g.float() * 2.0 ** power).half()
    _check(_step(q, k, v, g, data, causal=causal), _definition(q, k, v, g, lens, causal, dim ** -0.5))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shuffled", [False, True])
@pytest.mark.parametrize("lens,dim", [([700], 16), ([40, 64, 3], 32), ([2048], 64), ([2300, 1, 300], 128)])
def test_gradients_scale_with_the_outputs_gradient(lens, dim, shuffled, causal):
    """The gradients of 2^-p g are 2^-p times those of g.  Both are one sum in 32 bits up to a power of two, rounded to
    fp16: half a step each, and the smallest step for the small one."""
    ids, data = _plan(lens, shuffled, 4)
    q, k, v, _ = _inputs(sum(lens), 4, 2, dim, torch.float16, dim)
    gen = torch.Generator(device=DEV).manual_seed(1)
    g = torch.randint(-64, 65, (sum(lens), 4, dim), generator=gen, device=DEV).half() / 64
    full = _step(q, k, v, g, data, causal=causal)
    for p in (6, 10, 14):
        small = g * 2.0 ** -p
        assert torch.equal(small.double(), g.double() * 2.0 ** -p)
        got = _step(q, k, v, small, data, causal=causal)
        for name, a, b in zip(("g_q", "g_k", "g_v"), got[1:], full[1:]):
            off = (a.double() - b.double() * 2.0 ** -p).abs()
            bound = 2 * (H + 2 ** -20) * b.double().abs() * 2.0 ** -p + STEP * (1 + 2.0 ** -p)
            worst = float((off / bound).max())
            assert worst <= 1.0, f"2^-{p} {name}: {worst:.3g} of the bound"


@pytest.mark.parametrize("lens,dim", [([60, 64], 32), ([700], 16), ([900], 64)])
def test_large_gradients_in_other_segments(lens, dim):
    """Gradients near fp16's limit in one half of the segments, small ones in the other: each keeps its own precision."""
    ids, data = _plan([*lens, *lens], False)
    n = sum(lens)
    q, k, v, g = _inputs(2 * n, 2, 2, dim, torch.float16, 8)
    g[:n] = (g[:n].float() * 2.0 ** -12).half()
    g[n:] = (g[n:].float() * 8192).clamp(-60000, 60000).half()
    q[n:], k[n:] = q[n:] / 64, k[n:] / 64
    _check(_step(q, k, v, g, data), _definition(q, k, v, g, [*lens, *lens], False, dim ** -0.5))


@pytest.mark.parametrize("lens,dim", SHAPES)
def test_zeros_and_infinities(lens, dim):
    """No row has a largest value to go by: gradients are 0, not NaN."""
    ids, data = _plan(lens + lens, False)
    n = sum(lens)
    q, k, v, g = _inputs(2 * n, 4, 2, dim, torch.float16, 3)
    zero = torch.zeros_like
    for got in (_step(q, k, v, zero(g), data), _step(q, k, v, g, data, scale=0.0)):
        assert (got[1] == 0).all() and (got[2] == 0).all()
    assert (_step(q, k, v, zero(g), data)[3] == 0).all()
    got = _step(q, k, zero(v), g, data)
    assert (got[0] == 0).all() and (got[1] == 0).all() and (got[2] == 0).all() and got[3].isfinite().all()


@pytest.mark.parametrize("lens,dim", SHAPES)
def test_infinities_in_other_segments(lens, dim):
    ids, data = _plan(lens + lens, False)
    n = sum(lens)
    q, k, v, g = _inputs(2 * n, 2, 2, dim, torch.float16, 3)
    g = (g.float() * 2.0 ** -10).half()
    want = [(value[:n], bound[:n]) for value, bound in _definition(q, k, v, g, lens + lens, False, dim ** -0.5)]
    for i in (2, 3):
        ill = [q, k, v, g]
        ill[i] = ill[i].clone()
        ill[i][n:] = float("inf")
        _check([x[:n] for x in _step(*ill, data)], want)


def test_captured_and_on_another_stream():
    lens = [70, 200, 33, 600]
    ids, data = _plan(lens, True, 2)
    inputs = _inputs(sum(lens), 4, 2, 64, torch.float16, 4)
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        held = [torch.zeros_like(x) for x in inputs]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = _step(*held, data, causal=True)
        graphs.append((graph, held, outs))
    for seed, power in ((4, 0), (5, -12), (6, 3)):
        q, k, v, g = _inputs(sum(lens), 4, 2, 64, torch.float16, seed)
        new = [q, k, v, (g.float() * 2.0 ** power).half()]
        want = _step(*new, data, causal=True)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = _step(*new, data, causal=True)
        torch.cuda.current_stream().wait_stream(side)
        for graph, held, _ in graphs:
            for a, b in zip(held, new):
                a.copy_(b)
            graph.replay()
        torch.cuda.synchronize()
        for got in (other, *(outs for _, _, outs in graphs)):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
