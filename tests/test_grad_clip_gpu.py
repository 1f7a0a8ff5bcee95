"""The norm over many tensors and clipping by it, against a statement in 64 bits."""
import math

import pytest
import torch

from torchex_b200 import clip_grad_norm_, clip_grads, grad_norm

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _tensors(sizes, dtype, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=DEV) * scale).to(dtype) for n in sizes]


def _norm64(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


# Squares of eight values are added in fp32 (nine roundings of at most 2^-24 each, of positive terms) and the
# rest in fp64: the sum is off by at most 9 * 2^-24, its root by half of that, the rounding to fp32 adds 2^-24.
NORM_TOL = 5.5 * 2 ** -24


def _check_clipped(grads, outs, max_norm, norm):
    want = _norm64(grads)
    assert abs(norm.item() - want) <= NORM_TOL * want
    coef = min(1.0, max_norm / (want + 1e-6))
    for x, y in zip(grads, outs):
        ref = x.double() * coef
        half = torch.finfo(y.dtype).eps / 2
        tiny = torch.finfo(y.dtype).smallest_normal * half * 2
        # norm, the addition and the division of the coefficient, the product; then the output's half step
        assert ((y.double() - ref).abs() <= ref.abs() * (half + NORM_TOL + 4 * 2 ** -24) + tiny).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [
    (1,), (7,), (8,), (9, 1, 2), (16_384,), (16_383, 16_385, 0, 5), (100_000, 3, 70_001, 128, 128 * 16),
    (0,), tuple(range(1, 66)), tuple(100 + i for i in range(300)), tuple(1 + i % 7 for i in range(2100)), (6_000_001,),
])
def test_norm_and_clipping(dtype, sizes):
    grads = _tensors(sizes, dtype, len(sizes))
    want = _norm64(grads)
    assert abs(grad_norm(grads).item() - want) <= NORM_TOL * want
    kept = [x.clone() for x in grads]
    for factor in (0.3, 2.0):
        outs, norm = clip_grads(grads, factor * want)
        assert all(o.dtype == dtype and o.shape == x.shape for o, x in zip(outs, grads))
        _check_clipped(grads, outs, factor * want, norm)
        assert all(torch.equal(x, k) for x, k in zip(grads, kept))  # inputs stay
        wide = [torch.empty_like(x, dtype=torch.float32) for x in grads]
        got, norm2 = clip_grads(grads, factor * want, out=wide)
        assert torch.equal(norm, norm2) and all(a is b or a.data_ptr() == b.data_ptr() for a, b in zip(got, wide))
        _check_clipped(grads, wide, factor * want, norm2)
        own = [x.clone() for x in grads]
        clip_grads(own, factor * want, out=own)
        assert all(torch.equal(a, b) for a, b in zip(own, outs))  # in place: the same bits
        if factor > 1:
            assert all(torch.equal(a, b) for a, b in zip(own, grads))


@pytest.mark.parametrize("dtype", TYPES)
def test_views_that_start_anywhere_and_permuted_ones(dtype):
    base = _tensors((40_000,), dtype)[0]
    grads = [base[i * 9_000 + i:(i + 1) * 9_000 - 3 * i] for i in range(4)]
    outs = [torch.empty(40_000, device=DEV, dtype=dtype)[j:j + g.numel()] for j, g in zip((1, 0, 5, 8), grads)]
    got, norm = clip_grads(grads, 1.0, out=outs)
    _check_clipped(grads, outs, 1.0, norm)
    x = _tensors((6000,), dtype, 2)[0].view(10, 20, 30).permute(2, 0, 1)
    (y,), norm = clip_grads([x], 2.0)
    assert y.stride() == x.stride()
    _check_clipped([x], [y], 2.0, norm)
    x.copy_(torch.ones_like(x))
    around = base.clone()
    clip_grads([around[101:2003]], 1e-3, out=[around[101:2003]])  # neighbours stay as they were
    assert torch.equal(around[:101], base[:101]) and torch.equal(around[2003:], base[2003:])


def test_mixed_types_in_one_list():
    grads = [t for d in TYPES for t in _tensors((1000, 17, 33_000), d, 3)]
    outs, norm = clip_grads(grads, 5.0)
    _check_clipped(grads, outs, 5.0, norm)


def test_values_whose_squares_leave_the_range_of_32_bits():
    for scale in (1e-30, 3e-23, 1e-19, 1e19, 1e30):
        (x,) = _tensors((50_001,), torch.float32, 4, scale)
        want = _norm64([x])
        assert abs(grad_norm([x]).item() - want) <= NORM_TOL * want
        if scale > 1:
            (y,), norm = clip_grads([x], 1.0)
            _check_clipped([x], [y], 1.0, norm)
    mixed = torch.cat([torch.zeros(100, device=DEV), torch.full((9,), 1e-25, device=DEV), torch.zeros(5000, device=DEV)])
    assert abs(grad_norm([mixed]).item() - 3e-25) <= 3e-25 * (NORM_TOL + 2 ** -22)
    assert grad_norm([torch.full((2,), 3e38, device=DEV)]).item() == math.inf  # the norm itself overflows
    assert grad_norm([torch.zeros(12345, device=DEV)]).item() == 0.0


def test_many_values_do_not_drift():
    """2^27 equal values: their squares add up exactly in 64 bits, to 2^25.  Its root 2^12.5 has no
    exact 32-bit form, so the result is the 32-bit value nearest to it."""
    x = torch.full((1 << 27,), 0.5, device=DEV, dtype=torch.bfloat16)
    assert grad_norm([x]).item() == torch.tensor(math.sqrt((1 << 27) * 0.25), dtype=torch.float32).item()


@pytest.mark.parametrize("dtype", TYPES)
def test_non_finite_values(dtype):
    x, y = torch.ones(100, device=DEV, dtype=dtype), torch.ones(30, device=DEV, dtype=dtype)
    x[77] = float("inf")
    outs, norm = clip_grads([x, y], 1.0)
    assert norm.item() == math.inf and outs[0][77].isnan() and outs[0][:77].count_nonzero() == 0
    assert outs[1].count_nonzero() == 0
    x[3] = float("nan")
    outs, norm = clip_grads([x, y], 1.0)
    assert norm.isnan() and outs[0].isnan().all() and outs[1].isnan().all()
    params = [torch.nn.Parameter(torch.zeros(100, device=DEV)), torch.nn.Parameter(torch.zeros(30, device=DEV))]
    for bad in (float("inf"), float("nan")):  # the same as torch's own
        for p, q in zip(params, (x, y)):
            p.grad = q.float().nan_to_num(nan=bad, posinf=bad)
        ref = [torch.nn.Parameter(p.detach().clone()) for p in params]
        for r, p in zip(ref, params):
            r.grad = p.grad.clone()
        want, got = torch.nn.utils.clip_grad_norm_(ref, 1.0), clip_grad_norm_(params, 1.0)
        assert torch.equal(want.isnan(), got.isnan()) and torch.equal(want.isinf(), got.isinf())
        for r, p in zip(ref, params):
            assert torch.equal(r.grad.isnan(), p.grad.isnan())
            assert torch.equal(r.grad.nan_to_num(), p.grad.nan_to_num())


def test_parameters_in_place():
    m = torch.nn.Sequential(torch.nn.Linear(37, 64), torch.nn.Linear(64, 5), torch.nn.Linear(5, 5)).to(DEV)
    m[:2](torch.randn(9, 37, device=DEV)).square().sum().backward()  # the last layer has no gradient
    before = [p.grad.clone() for p in m[:2].parameters()]
    versions = [p.grad._version for p in m[:2].parameters()]
    norm = clip_grad_norm_(m.parameters(), 0.5)
    _check_clipped(before, [p.grad for p in m[:2].parameters()], 0.5, norm)
    assert all(p.grad._version > v for p, v in zip(m[:2].parameters(), versions))
    assert abs(grad_norm([p.grad for p in m[:2].parameters()]).item() - 0.5) < 1e-5
    one = torch.nn.Parameter(torch.zeros(3, device=DEV))
    one.grad = torch.full((3,), 2.0, device=DEV)
    assert clip_grad_norm_(one, 100.0).item() == pytest.approx(math.sqrt(12)) and (one.grad == 2).all()


def test_refusals():
    x, y = torch.ones(100, device=DEV), torch.ones(50, device=DEV)
    p = torch.nn.Parameter(x)
    p.grad = x
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grad_norm_([p, p], 1.0)
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([x, y], 1.0, out=[x, x[20:70]])
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([x[:50], y], 1.0, out=[x[10:60], y])
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([x[:50], y], 1.0, out=[y, x[:50]])
    assert (x == 1).all() and (y == 1).all()
    with pytest.raises(RuntimeError, match="gaps or overlaps"):
        grad_norm([x[::2]])
    with pytest.raises(RuntimeError, match="gaps or overlaps"):
        grad_norm([x[:1].expand(5)])
    with pytest.raises(RuntimeError, match="another shape"):
        clip_grads([x], 1.0, out=[y])
    with pytest.raises(RuntimeError, match="other strides"):
        clip_grads([x.view(10, 10)], 1.0, out=[torch.empty(10, 10, device=DEV).t()])
    with pytest.raises(RuntimeError, match="dtype of its gradient or float32"):
        clip_grads([x], 1.0, out=[x.half()])
    with pytest.raises(RuntimeError, match="2 tensors for 1"):
        clip_grads([x], 1.0, out=[x, y])
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        grad_norm([x.double()])
    with pytest.raises(RuntimeError, match="sparse"):
        grad_norm([x.to_sparse()])
    with pytest.raises(RuntimeError, match="CUDAtensor"):
        grad_norm([x, torch.ones(3)])
    assert grad_norm([x, x]).item() == pytest.approx(math.sqrt(200))  # reading twice is fine


def test_streams_and_graph_replay():
    sizes = (30_000, 5, 77, 100_001)
    grads = _tensors(sizes, torch.bfloat16, 6)
    want, norm = clip_grads(grads, 1.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, n2 = clip_grads(grads, 1.5)
    side.synchronize()
    assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(want, got))
    held = [[torch.zeros_like(g) for g in grads] for _ in range(2)]
    graphs, results = [], []
    for h in held:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(clip_grads(h, 1.5))
    for h, scale in zip(held, (1.0, 2.0)):
        for a, b in zip(h, grads):
            a.copy_(b * scale)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for h, (outs, n) in zip(held, results):
        ref, nr = clip_grads(h, 1.5)
        assert torch.equal(n, nr) and all(torch.equal(a, b) for a, b in zip(outs, ref))


def test_tensors_that_require_a_gradient():
    """Neither result has a gradient, so it is not taken from tensors that would record one."""
    p = torch.nn.Parameter(torch.full((16,), 2.0, device=DEV))
    x = torch.ones(16, device=DEV)
    for call in (lambda: grad_norm([p]), lambda: clip_grads([p], 1.0), lambda: clip_grads([x], 1.0, out=[p]),
                 lambda: grad_norm([p * 2])):
        with pytest.raises(RuntimeError, match="not differentiable"):
            call()
    assert (p == 2).all()
    with torch.no_grad():
        assert grad_norm([p]).item() == 8.0
    p.grad, = torch.autograd.grad((p * p).sum(), p, create_graph=True)  # 2 p
    assert p.grad.requires_grad
    assert clip_grad_norm_(p, 8.0).item() == 16.0
    assert torch.allclose(p.grad, torch.full_like(x, 2.0))


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        x, y = torch.ones(3, device=DEV), torch.empty(3, device=DEV)
        dual = fwd.make_dual(torch.ones(3, device=DEV), torch.ones(3, device=DEV))
        for call in (lambda: grad_norm([x, dual]), lambda: clip_grads([dual], 1.0), lambda: clip_grads([x, dual], 1.0, out=[y, x]),
                     lambda: clip_grads([x], 1.0, out=[dual])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert float(grad_norm([x])) == pytest.approx(3 ** 0.5)
