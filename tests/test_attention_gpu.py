"""Attention within segments against its definition in 64 bits.

Every comparison is by a bound that follows from the roundings of the operator.  With h the half step
of the tensors' type (2^-8 for bf16, 2^-11 for fp16) and e the relative error of a probability before it
is rounded (scores and exponentials in 32 bits), an output is off by at most
    h |o| + (h + e) sum_j p_j |v_j|
and the gradients by the same reasoning, term by term (``_bounds``).
"""
import pytest
import torch

from torchex_b200 import ScatterData, scatter_mean, segment_attention

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16]


def _plan(lens, shuffled, seed=0):
    ids = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    if shuffled:
        ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(seed))]
    ids = ids.to(DEV)
    return ids, ScatterData(ids, torch.tensor(lens, device=DEV))


def _inputs(n, heads, kv_heads, dim, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(n, h, dim, generator=g, device=DEV).to(dtype) for h in (heads, kv_heads, kv_heads, heads)]


def _definition(q, k, v, g, ids, segments, scale, causal, cap, slopes):
    """Outputs and gradients in 64 bits, and the bound of each: [(value, bound)] for o, gq, gk, gv."""
    h = torch.finfo(q.dtype).eps / 2
    # half of the type's smallest step; and exponentials below 2^-126 become 0, so that a probability may be off by that
    # much before it is rounded, and a gradient of a score by that much times |g v - delta| scale (added below)
    under = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps / 2 + 2 ** -126
    q, k, v, g = (x.double() for x in (q, k, v, g))
    group = q.shape[1] // k.shape[1]
    found = [[torch.zeros_like(x), torch.zeros_like(x)] for x in (q, q, k, v)]
    for s in range(segments):
        rows = (ids == s).nonzero()[:, 0]
        n = rows.numel()
        if n == 0:
            continue
        qs, ks, vs, gs = (x[rows].transpose(0, 1) for x in (q, k, v, g))
        ks, vs = ks.repeat_interleave(group, 0), vs.repeat_interleave(group, 0)
        raw = qs @ ks.mT * scale
        size = qs.abs() @ ks.abs().mT * abs(scale)
        d_score = (qs.shape[2] + 4) * 2 ** -24 * size  # products exact, their sum and the scaling in 32 bits
        x, slope = raw, torch.ones_like(raw)
        if cap:
            t = torch.tanh(raw / cap)
            x, slope = cap * t, 1 - t * t
            d_score = d_score + cap * 2 ** -21        # tanh from one exponential and one division
        at = torch.arange(n, device=DEV)
        if slopes is not None:
            bias = slopes.double()[:, None, None] * (at[:, None] - at).abs()
            x, d_score = x - bias, d_score + 2 ** -23 * bias
        d_score = d_score + 2 ** -22 * x.abs()        # to units of log2, and the subtraction of the maximum
        if causal:
            x = x.masked_fill(at > at[:, None], float("-inf"))
        p = torch.softmax(x, -1)
        seen = (p > 0) if not causal else (at <= at[:, None]).expand_as(p)
        d_score = torch.where(seen, d_score, 0.0)
        # relative error of a probability: its own score, the weighted mean of the others, two exponentials, sums
        e = d_score + (p * d_score).sum(-1, keepdim=True) + (n + 16) * 2 ** -24
        e = torch.expm1(2 * e)
        o = p @ vs
        bound_o = h * o.abs() + (p * (h + e)) @ vs.abs() + under * (seen.double() @ vs.abs() + 1)
        dp = gs @ vs.mT
        delta = (gs * o).sum(-1, keepdim=True)
        d_dp = (qs.shape[2] + 2) * 2 ** -24 * (gs.abs() @ vs.abs().mT)
        d_delta = (gs.abs() * bound_o).sum(-1, keepdim=True) + (qs.shape[2] + 2) * 2 ** -24 * (gs * o).abs().sum(-1, keepdim=True)
        ds = p * (dp - delta) * slope * scale
        d_ds = p * (d_dp + d_delta) * abs(scale) + (e + h + 2 ** -22) * (ds.abs() + p * (d_dp + d_delta) * abs(scale)) + under * seen
        d_ds = d_ds + 2 ** -126 * ((dp - delta).abs() + d_dp + d_delta) * slope * abs(scale) * seen
        if cap:
            d_ds = d_ds + p * ((dp - delta).abs() + d_dp + d_delta) * abs(scale) * 2 ** -19  # 1 - t^2 from t
        d_p = p * (h + e) + under * seen
        sums = (n + 4) * 2 ** -24
        terms = [(o, bound_o),
                 (ds @ ks, d_ds @ ks.abs() + (sums + 0.0) * (ds.abs() @ ks.abs())),
                 (ds.mT @ qs, d_ds.mT @ qs.abs() + sums * (ds.abs().mT @ qs.abs())),
                 (p.mT @ gs, d_p.mT @ gs.abs() + sums * (p.mT @ gs.abs()))]
        for i, (value, bound) in enumerate(terms):
            if i >= 2:  # shared heads: one gradient
                value, bound = (y.unflatten(0, (-1, group)).sum(1) for y in (value, bound))
            if i >= 1:
                bound = bound + h * value.abs() + under
            found[i][0][rows], found[i][1][rows] = value.transpose(0, 1), bound.transpose(0, 1)
    return found


def _step(q, k, v, g, data, **kw):
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out = segment_attention(q, k, v, data, **kw)
    return [out.detach(), *torch.autograd.grad(out, (q, k, v), g)]


def _check(got, want, rows=None, label=""):
    for name, y, (value, bound) in zip(("out", "g_q", "g_k", "g_v"), got, want):
        assert y.shape == value.shape
        off = (y.double() - value).abs()
        if rows is not None:
            off, bound = off[rows], bound[rows]
        bad = ~(off <= bound)
        assert not bad.any(), f"{label} {name}: {int(bad.sum())} of {bad.numel()}, worst {float((off / bound).nan_to_num(9e9).max()):.3g} of the bound"


LENS = {
    "one": [1], "ones": [1] * 130, "tile": [64], "tile and one": [65], "mixed": [63, 1, 64, 129, 2, 30],
    "gaps": [5, 0, 7, 0, 0, 70, 0], "short": [3 + 5 * i % 17 for i in range(60)], "long": [777], "two long": [513, 3, 260],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 8), (2, 1, 16), (4, 4, 24), (3, 3, 32), (6, 2, 40), (2, 2, 64), (2, 1, 80),
                                                (2, 2, 128)])
@pytest.mark.parametrize("lens", LENS)
def test_outputs_and_gradients(dtype, causal, heads, kv_heads, dim, lens):
    lens = LENS[lens]
    shuffled = (dim // 8) % 2 == 0
    ids, data = _plan(lens, shuffled, dim)
    q, k, v, g = _inputs(sum(lens), heads, kv_heads, dim, dtype, dim + len(lens))
    scale = dim ** -0.5
    want = _definition(q, k, v, g, ids, len(lens), scale, causal, 0.0, None)
    got = _step(q, k, v, g, data, causal=causal)
    _check(got, want)
    data.max_cnt  # from here on the plan's statistics are known to the host
    again = _step(q, k, v, g, data, causal=causal)
    _check(again, want)
    third = _step(q, k, v, g, data, causal=causal)
    assert all(torch.equal(a, b) for a, b in zip(again, third))  # reproducible to the bit


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("cap,with_slopes", [(5.0, False), (50.0, True), (0.0, True)])
@pytest.mark.parametrize("dim", [16, 40, 64, 128])
def test_capped_scores_and_distance(dtype, causal, cap, with_slopes, dim):
    lens = [70, 1, 200, 9, 33]
    ids, data = _plan(lens, True, 3)
    q, k, v, g = _inputs(sum(lens), 4, 2, dim, dtype, 7)
    slopes = torch.tensor([0.5, 0.1, 0.02, 0.0], device=DEV) if with_slopes else None
    scale = 3.0 * dim ** -0.5
    want = _definition(q, k, v, g, ids, len(lens), scale, causal, cap, slopes)
    _check(_step(q, k, v, g, data, scale=scale, causal=causal, softcap=cap, slopes=slopes), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dtype):
    """Scores of some hundreds: one key takes all the weight; capped ones go to the cap."""
    lens = [100, 40]
    ids, data = _plan(lens, False)
    q, k, v, g = _inputs(140, 2, 2, 64, dtype, 5)
    q, k = q * 8, k * 8
    for cap in (0.0, 20.0):
        want = _definition(q, k, v, g, ids, 2, 0.5, False, cap, None)
        _check(_step(q, k, v, g, data, scale=0.5, softcap=cap), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, dim, causal):
    """Segments 1 and 3 hold NaN and infinities in every tensor; with `causal`, so does the last row of 4."""
    lens = [40, 20, 90, 5, 70, 200]
    ids, data = _plan(lens, dim == 64, 1)
    for known in (False, True):
        if known:
            data.max_cnt
        q, k, v, g = _inputs(sum(lens), 4, 2, dim, dtype, 11)
        clean = [x.clone() for x in (q, k, v, g)]
        ill = (ids == 1) | (ids == 3)
        for i, x in enumerate((q, k, v, g)):
            x[ill] = (float("nan"), float("inf"), float("-inf"))[i % 3]
        last = (ids == 4).nonzero()[-1, 0]
        if causal:
            for x in (k, v):
                x[last] = float("nan")
        want = _definition(*clean, ids, len(lens), dim ** -0.5, causal, 0.0, None)
        got = _step(q, k, v, g, data, causal=causal)
        rows = ~ill
        if not causal:
            _check(got, want, rows)
            continue
        before = rows.clone()
        before[last] = False
        _check(got[:1], want[:1], before)      # rows in front of the last one do not see it
        _check(got[1:2], want[1:2], before)
        _check(got[2:], want[2:], rows & (ids != 4))  # its own gradients reach the keys that it sees
        assert got[0][last].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_non_finite_values_that_are_seen(dtype):
    """An infinite value reaches the rows of its segment, in its column."""
    lens = [70, 70]
    ids, data = _plan(lens, False)
    q, k, v, g = _inputs(140, 1, 1, 32, dtype, 2)
    v[75, 0, 3] = float("inf")
    out = segment_attention(q, k, v, data)
    assert (out[70:, 0, 3] == float("inf")).all()
    out[70:, 0, 3] = 0
    assert out.isfinite().all()
    k[75, 0, 0] = float("nan")
    out = segment_attention(q, k, v, data)
    assert out[70:].isnan().all() and out[:70].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_expanded_gradients(dtype):
    lens = [30, 100]
    ids, data = _plan(lens, True, 9)
    n, heads, dim = 130, 4, 32
    fused = torch.randn(n, 3, heads, dim, device=DEV).to(dtype)
    g = torch.randn(n, 1, dim, device=DEV).to(dtype).expand(n, heads, dim)
    want = _definition(fused[:, 0], fused[:, 1], fused[:, 2], g, ids, 2, dim ** -0.5, False, 0.0, None)
    _check(_step(fused[:, 0], fused[:, 1], fused[:, 2], g, data), want, label="fused")
    by_head = torch.randn(3, heads, n, dim, device=DEV).to(dtype).transpose(1, 2)
    g = torch.ones((), device=DEV, dtype=dtype).expand(n, heads, dim)
    want = _definition(by_head[0], by_head[1], by_head[2], g, ids, 2, dim ** -0.5, False, 0.0, None)
    _check(_step(by_head[0], by_head[1], by_head[2], g, data), want, label="by head")
    odd = torch.randn(n * heads * dim + 1, device=DEV).to(dtype)[1:].view(n, heads, dim)  # off every 16-byte boundary
    last = torch.randn(n, dim, heads, device=DEV).to(dtype).transpose(1, 2)               # head dimension not contiguous
    want = _definition(odd, last, odd, last, ids, 2, dim ** -0.5, False, 0.0, None)
    _check(_step(odd, last, odd, last, data), want, label="copied")


def test_gradients_follow_differences():
    """(L(x + t d) - L(x - t d)) / 2t against <gradient, d>, L = <g, out>, on values where every input of the
    difference is exact (small integers over 64) and bf16 rounding of the two outputs is counted."""
    lens = [20, 45]
    ids, data = _plan(lens, False)
    gen = torch.Generator(device=DEV).manual_seed(3)
    q, k, v, d = (torch.randint(-32, 33, (65, 2, 16), generator=gen, device=DEV).to(torch.float16) / 64 for _ in range(4))
    g = torch.randint(-32, 33, (65, 2, 16), generator=gen, device=DEV).to(torch.float16) / 64
    grads = _step(q, k, v, g, data)[1:]
    t = 0.125
    for i, grad in enumerate(grads):
        plus, minus = [q, k, v], [q, k, v]
        plus[i], minus[i] = plus[i] + t * d, minus[i] - t * d
        a, b = (segment_attention(*x, data).double() for x in (plus, minus))
        slope = float(((a - b) * g.double()).sum() / (2 * t))
        rounding = float(((a.abs() + b.abs()) * g.double().abs()).sum()) * 2 ** -10 / (2 * t)
        right = float((grad.double() * d.double()).sum())
        size = float((grad.double().abs() * d.double().abs()).sum())
        # third-order terms of the difference: t^2 / 6 times a third derivative; scores are below 1 in size, so it is
        # within 4 (|scale d|^3 n) of 0 for q and k, and none for v, in which the output is linear
        third = 0.0 if i == 2 else t * t * size
        assert abs(slope - right) <= rounding + third + size * 2 ** -9


def test_rows_and_heads_beyond_32_bit_offsets():
    n, heads, dim = 150_000, 112, 128  # 2.15e9 values
    q = torch.zeros(n, heads, dim, device=DEV, dtype=torch.bfloat16)
    k, v = (torch.randn(n, 1, dim, device=DEV).to(torch.bfloat16) for _ in range(2))
    ids = torch.arange(n, device=DEV) // 3
    data = ScatterData(ids, torch.full((n // 3,), 3, device=DEV))
    out = segment_attention(q, k, v, data)  # zero queries: the mean of the values
    mean = scatter_mean(v[:, 0].float().contiguous(), data)
    for row in (0, 1, n - 1, n - 2, n // 2):
        want = mean[ids[row]].expand(heads, dim)
        assert ((out[row].float() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -7 * v[3 * int(ids[row]):3 * int(ids[row]) + 3, 0].float().abs().mean(0)).all()


def test_streams_graphs_and_an_eager_graph_beside():
    lens = [70, 200, 33]
    ids, data = _plan(lens, True, 2)
    data.max_cnt
    q, k, v, g = _inputs(sum(lens), 4, 2, 64, torch.bfloat16, 4)
    want = _step(q, k, v, g, data, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(q, k, v, g, data, causal=True)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = []
    for _ in range(2):
        ins = [torch.zeros_like(x) for x in (q, k, v, g)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = _step(*ins, data, causal=True)
        held.append((graph, ins, outs))
    for seed in (4, 5):
        new = _inputs(sum(lens), 4, 2, 64, torch.bfloat16, seed)
        want = _step(*new, data, causal=True)
        for graph, ins, _ in held:
            for a, b in zip(ins, new):
                a.copy_(b)
        for graph, *_ in held:
            graph.replay()
        torch.cuda.synchronize()
        for _, _, outs in held:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("lens", [[30, 40, 7], [300, 200]])
def test_gradients_that_are_not_wanted(lens):
    ids, data = _plan(lens, False)
    q, k, v, g = _inputs(sum(lens), 2, 1, 64, torch.bfloat16, 6)
    full = _step(q, k, v, g, data)
    for wanted in ((0,), (1,), (2,), (0, 2)):
        ins = [x.detach().clone().requires_grad_(i in wanted) for i, x in enumerate((q, k, v))]
        out = segment_attention(*ins, data)
        grads = torch.autograd.grad(out, [ins[i] for i in wanted], g)
        assert all(torch.equal(a, full[1 + i]) for i, a in zip(wanted, grads))


def test_empty_batch_and_refusals():
    data = ScatterData(torch.zeros(0, dtype=torch.int64, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV))
    e = torch.zeros(0, 2, 16, device=DEV, dtype=torch.float16, requires_grad=True)
    out = segment_attention(e, e, e, data)
    assert out.shape == (0, 2, 16)
    out.sum().backward()
    ids, data = _plan([4, 6], False)
    q = torch.zeros(10, 4, 16, device=DEV, dtype=torch.bfloat16)
    kv = q[:, :2]
    for message, args, kw in [
            ("bfloat16 or float16", (q.float(), kv, kv), {}), ("another dtype", (q, kv.half(), kv), {}),
            ("multiple of 8", (q[..., :12], kv[..., :12], kv[..., :12]), {}),
            ("multiple of 8", tuple(torch.zeros(10, 1, 136, device=DEV, dtype=torch.bfloat16) for _ in range(3)), {}),
            ("evenly", (q[:, :3], kv, kv), {}), ("different numbers", (q, kv, q), {}), ("built for", (q[:9], kv[:9], kv[:9]), {}),
            ("head dimension", (q, kv[..., :8], kv), {}), ("softcap", (q, kv, kv), {"softcap": -1.0}),
            ("softcap", (q, kv, kv), {"softcap": float("inf")}), ("scale", (q, kv, kv), {"scale": float("nan")}),
            ("per query head", (q, kv, kv), {"slopes": torch.zeros(2, device=DEV)}),
            ("dtype", (q, kv, kv), {"slopes": torch.zeros(4, device=DEV, dtype=torch.float16)}),
            ("no gradient", (q, kv, kv), {"slopes": torch.zeros(4, device=DEV, requires_grad=True)}),
            ("CUDAtensor", (q.cpu(), kv, kv), {})]:
        with pytest.raises(RuntimeError, match=message):
            segment_attention(*args, data, **kw)
    x = q.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(segment_attention(x, kv, kv, data).sum(), x, create_graph=True)
    assert not segment_attention(x.detach(), kv, kv, data).requires_grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,dim", [([70, 1, 200], 16), ([200, 150], 64), ([200, 150], 128)])
def test_cap_far_above_the_scores(dtype, lens, dim):
    """A cap of a million leaves scores of a few units what they are (cap tanh(x / cap) = x to 1e-11), so the formulas
    without a cap hold.  Beside the roundings that their bound counts for a score x, (dim + 4 + 4) 2^-24 |x| at least,
    the cap has nine: two factors, two products with them, five of the series; so twice the bound is enough, and a
    hundredth for its curvature."""
    ids, data = _plan(lens, True, 3)
    q, k, v, g = _inputs(sum(lens), 4, 2, dim, dtype, 7)
    want = [(value, 2.01 * bound) for value, bound in _definition(q, k, v, g, ids, len(lens), dim ** -0.5, False, 0.0, None)]
    _check(_step(q, k, v, g, data, softcap=1e6), want)


def test_caps_out_of_range_are_refused():
    ids, data = _plan([4, 6], False)
    q = torch.zeros(10, 4, 16, device=DEV, dtype=torch.bfloat16)
    for cap in (1e-300, 1e-42, 3e38):
        with pytest.raises(RuntimeError, match="softcap"):
            segment_attention(q, q, q, data, softcap=cap)


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    ids, data = _plan([4, 6], False)
    q = torch.zeros(10, 4, 16, device=DEV, dtype=torch.bfloat16)
    with fwd.dual_level():
        for i in range(3):
            args = [q, q, q]
            args[i] = fwd.make_dual(q, torch.ones_like(q))
            with pytest.raises(RuntimeError, match="forward-mode"):
                segment_attention(*args, data)


@pytest.mark.parametrize("n,heads", [(70, 1), (1, 3), (1, 1)])
def test_strides_of_axes_of_one(n, heads):
    """The stride of an axis of size one says nothing, whatever it is."""
    ids, data = _plan([n], False)
    q, k, v, g = _inputs(n, heads, heads, 16, torch.bfloat16, 4)
    want = _step(q, k, v, g, data)

    def odd(x):
        strides = [1 if size == 1 else stride for size, stride in zip(x.shape, x.stride())]
        y = x.as_strided(x.shape, strides)
        assert y.is_contiguous() and torch.equal(x, y)
        return y

    for a, b in zip(_step(odd(q), odd(k), odd(v), odd(g), data), want):
        assert torch.equal(a, b)


def test_forward_mode_is_refused_for_slopes_and_gradients():
    import torch.autograd.forward_ad as fwd

    ids, data = _plan([4, 6], False)
    q = torch.zeros(10, 4, 16, device=DEV, dtype=torch.bfloat16)
    x = q.clone().requires_grad_(True)
    out = segment_attention(x, q, q, data)
    slopes = torch.zeros(4, device=DEV)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            segment_attention(q, q, q, data, slopes=fwd.make_dual(slopes, torch.ones_like(slopes)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, x, fwd.make_dual(q, torch.ones_like(q)))
