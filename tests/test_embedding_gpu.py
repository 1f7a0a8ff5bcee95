"""Table lookup and its gradient against a plain statement in 64 bits."""
import math

import pytest
import torch

from torchex_b200 import ScatterData, _native, embedding, gather_back, scatter_sum

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _tokens(n, vocab, seed, kind="flat", id_dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if kind == "same":
        t = torch.full((n,), vocab // 2)
    elif kind == "zipf":
        t = (torch.pow(float(vocab), torch.rand(n, generator=g, dtype=torch.float64)) - 1).long().clamp(0, vocab - 1)
    else:
        t = torch.randint(0, vocab, (n,), generator=g)
    return t.to(DEV).to(id_dtype)


def _check(tokens, weight, g, scale, pad, out, g_weight):
    """|error| of the output: the half step of its type; of the gradient: that, and the additions in
    32 bits of a row's c terms, each off by at most 2^-24 of a partial sum <= sum |g|."""
    half = torch.finfo(weight.dtype).eps / 2
    tiny = torch.finfo(weight.dtype).smallest_normal * half * 2
    flat = tokens.reshape(-1).long()
    ok = (flat >= 0) & (flat < weight.shape[0])
    want = torch.zeros(flat.numel(), weight.shape[1], dtype=torch.float64, device=DEV)
    want[ok] = weight.detach().double()[flat[ok]] * scale
    got = out.detach().reshape(want.shape).double()
    assert ((got - want).abs() <= (half + 2 ** -23) * want.abs() + tiny).all()
    if g_weight is None:
        return
    if pad is not None:
        ok &= flat != pad
    rows = g.reshape(want.shape).double()[ok]
    total = torch.zeros(weight.shape, dtype=torch.float64, device=DEV).index_add_(0, flat[ok], rows) * scale
    size = torch.zeros(weight.shape, dtype=torch.float64, device=DEV).index_add_(0, flat[ok], rows.abs()) * abs(scale)
    count = torch.bincount(flat[ok], minlength=weight.shape[0]).double()[:, None]
    allowed = (half + 2 ** -23) * total.abs() + (count + 2) * 2 ** -24 * size + tiny
    if weight.dtype == torch.float32:  # error-free additions: second-order terms only
        allowed = 2 ** -22 * total.abs() + (count * 2 ** -24) ** 2 * size + tiny
    bad = (g_weight.double() - total).abs() > allowed
    assert not bad.any(), f"{int(bad.sum())} values outside the bound"


def _step(tokens, weight, g, scale=1.0, pad=None):
    w = weight.detach().requires_grad_(True)
    out = embedding(tokens, w, scale=scale, padding_idx=pad)
    assert out.shape == (*tokens.shape, weight.shape[1]) and out.dtype == weight.dtype
    (gw,) = torch.autograd.grad(out, w, g)
    assert gw.shape == weight.shape and gw.dtype == weight.dtype
    return out, gw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,dim,kind", [
    (1, 1, 1, "flat"), (1, 5000, 64, "flat"), (2, 3, 7, "same"), (31, 9, 8, "flat"), (64, 40, 33, "zipf"),
    (257, 1000, 16, "zipf"), (1000, 300, 515, "flat"), (4096, 4097, 128, "zipf"), (5000, 64, 260, "zipf"),
    (20_000, 2000, 24, "flat"), (9000, 70_000, 40, "zipf"), (3001, 5, 1024, "same"), (40_000, 7, 96, "zipf"),
    (140_001, 3000, 10, "zipf"), (33_000, 260, 2050, "zipf"),
])
def test_lookup_and_gradient(dtype, n, vocab, dim, kind):
    g0 = torch.Generator(device=DEV).manual_seed(n + dim)
    weight = torch.randn(vocab, dim, generator=g0, device=DEV).to(dtype)
    g = torch.randn(n, dim, generator=g0, device=DEV).to(dtype)
    tokens = _tokens(n, vocab, n, kind, torch.int32 if n % 2 else torch.int64)
    for scale, pad in ((1.0, None), (0.375, vocab // 2)):
        out, gw = _step(tokens, weight, g, scale, pad)
        _check(tokens, weight, g, scale, pad, out, gw)
        if pad is not None:
            assert (gw[pad] == 0).all()
    again = _step(tokens, weight, g, 0.375, vocab // 2)
    assert torch.equal(again[1], gw) and torch.equal(again[0], out)  # reproducible to the bit


@pytest.mark.parametrize("dtype", TYPES)
def test_scale_of_one_copies_every_value(dtype):
    weight = torch.tensor([float("nan"), float("inf"), float("-inf"), -0.0, 0.0, 1e-7, 6e-5, 1.5], device=DEV).to(dtype)[None]
    out = embedding(torch.zeros(3, dtype=torch.int64, device=DEV), weight)
    kind = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(out.view(kind), weight.expand(3, -1).contiguous().view(kind))


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_batches_and_shapes_of_tokens(dtype):
    weight = torch.randn(70_001, 12, device=DEV).to(dtype)
    for shape in ((0,), (3, 0), (2, 3, 4), ()):
        tokens = torch.ones(shape, dtype=torch.int64, device=DEV)
        out, gw = _step(tokens, weight, torch.ones(*shape, 12, device=DEV, dtype=dtype))
        assert out.shape == (*shape, 12)
        assert (gw[1] == tokens.numel()).all() and gw[:1].count_nonzero() == 0 and gw[2:].count_nonzero() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_non_finite_gradients_reach_their_own_row_only(dtype):
    tokens = torch.tensor([4, 1, 4, 2, 1, 0], device=DEV)
    weight = torch.zeros(6, 20, device=DEV, dtype=dtype)
    g = torch.ones(6, 20, device=DEV, dtype=dtype)
    g[0, 3], g[2, 4], g[1, 5], g[4, 5], g[3, 6] = float("nan"), float("inf"), float("inf"), float("-inf"), float("inf")
    _, gw = _step(tokens, weight, g, pad=2)
    assert gw[4, 3].isnan() and gw[4, 4] == float("inf") and gw[1, 5].isnan()
    gw[4, 3], gw[4, 4], gw[1, 5] = 2, 2, 2
    assert torch.equal(gw, torch.tensor([1, 2, 0, 0, 2, 0], device=DEV)[:, None].expand(6, 20).to(dtype))


def test_tokens_out_of_range_are_counted_and_left_out():
    before = _native.device_bad_indices()
    tokens = torch.tensor([0, -1, 3, 7, 2 ** 40, 3, -2 ** 62], device=DEV)
    weight = torch.randn(7, 36, device=DEV)
    g = torch.randn(7, 36, device=DEV)
    out, gw = _step(tokens, weight, g, 2.0)
    _check(tokens, weight, g, 2.0, None, out, gw)
    assert (out[[1, 3, 4, 6]] == 0).all()
    assert _native.device_bad_indices() == before + 8  # four tokens, forward and backward


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_offsets_and_expanded_gradients(dtype):
    n, vocab, dim = 300, 50, 24
    tokens = _tokens(2 * n, vocab, 1)[::2]
    base = torch.randn(dim, vocab, device=DEV).to(dtype)
    g = torch.randn(1, dim, device=DEV).to(dtype).expand(n, dim)
    out, gw = _step(tokens, base.t(), g, 0.5)
    _check(tokens, base.t(), g, 0.5, None, out, gw)
    for shift in (1, 2, 3, 4):  # rows that start off a 16-byte boundary
        w = torch.randn(vocab * dim + shift, device=DEV).to(dtype)[shift:].view(vocab, dim)
        gs = torch.randn(n * dim + shift, device=DEV).to(dtype)[shift:].view(n, dim)
        out, gw = _step(tokens, w, gs, 0.5)
        _check(tokens, w, gs, 0.5, None, out, gw)


def test_the_gradient_is_the_transpose_of_the_lookup():
    """<g, embedding(h)> = <g_w, h> for any h, and differences of the output follow it."""
    tokens = _tokens(500, 60, 3, "zipf")
    w = torch.randn(60, 17, device=DEV)
    g = torch.randn(500, 17, device=DEV)
    h = torch.randn(60, 17, device=DEV)
    _, gw = _step(tokens, w, g, 3.0)
    moved = (embedding(tokens, w + h, scale=3.0).double() - embedding(tokens, w - h, scale=3.0).double()) / 2
    left, right = (moved * g.double()).sum(), (gw.double() * h.double()).sum()
    size = float((moved.abs() * g.double().abs()).sum())
    assert abs(float(left - right)) <= 8 * 2 ** -24 * size  # rounding of w +- h, of two products and of gw


def test_table_beyond_32_bit_offsets():
    vocab, dim = 1_050_000, 2056  # 2.16e9 values
    weight = torch.empty(vocab, dim, device=DEV, dtype=torch.bfloat16)
    weight[:3] = 1.0
    weight[-3:] = torch.arange(dim, device=DEV).to(torch.bfloat16)
    tokens = torch.tensor([vocab - 1, 0, vocab - 2, 2], device=DEV)
    g = torch.randn(4, dim, device=DEV).to(torch.bfloat16)
    out, gw = _step(tokens, weight, g)
    assert torch.equal(out[0], weight[-1]) and torch.equal(out[2], weight[-2]) and (out[[1, 3]] == 1).all()
    assert torch.equal(gw[[vocab - 1, 0, vocab - 2, 2]], g)
    assert gw[3:vocab - 2].count_nonzero() == 0 and gw[vocab // 2 - 5:vocab // 2].count_nonzero() == 0


def test_matches_the_segment_operators_on_a_plan():
    """The lookup is gather_back, its gradient scatter_sum, for the plan of the same ids."""
    ids = _tokens(4000, 500, 9, "zipf")
    data = ScatterData(ids, torch.bincount(ids, minlength=500))
    table, g = torch.randn(500, 64, device=DEV), torch.randn(4000, 64, device=DEV)
    out, gw = _step(ids, table, g)
    assert torch.equal(out, gather_back(table, data))
    assert torch.allclose(gw, scatter_sum(g, data), rtol=2 ** -22, atol=0)


def test_streams_and_graph_replay():
    n, vocab, dim = 6000, 900, 64
    weight = torch.randn(vocab, dim, device=DEV).to(torch.bfloat16).requires_grad_(True)
    tokens, g = _tokens(n, vocab, 5, "zipf"), torch.randn(n, dim, device=DEV).to(torch.bfloat16)
    want = _step(tokens, weight, g, 2.0, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(tokens, weight, g, 2.0, 3)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn: each has workspaces of its own
        graph = torch.cuda.CUDAGraph()
        tok, gg = torch.zeros_like(tokens), torch.zeros_like(g)
        w = weight.detach().clone().requires_grad_(True)
        with torch.cuda.graph(graph):
            out = embedding(tok, w, scale=2.0, padding_idx=3)
            (gw,) = torch.autograd.grad(out, w, gg)
        graphs.append((graph, tok, gg, out, gw))
    for seed in (5, 6):
        tokens = _tokens(n, vocab, seed, "zipf")
        want = _step(tokens, weight, g, 2.0, 3)
        for graph, tok, gg, out, gw in graphs:
            tok.copy_(tokens)
            gg.copy_(g)
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, _, _, out, gw in graphs:
            assert torch.equal(out, want[0]) and torch.equal(gw, want[1])


def test_gradient_only_where_it_is_wanted():
    w = torch.randn(9, 4, device=DEV, requires_grad=True)
    tok = torch.tensor([1, 2], device=DEV)
    with torch.no_grad():
        assert not embedding(tok, w).requires_grad
    assert not embedding(tok, w.detach()).requires_grad
    with pytest.raises(RuntimeError, match="int32 or int64"):
        embedding(tok.float(), w)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        embedding(tok, w.detach().double())
    with pytest.raises(RuntimeError, match="CUDAtensor"):
        embedding(tok, torch.zeros(4, 4))
    out = embedding(tok, w).sum()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out, w, create_graph=True)
    assert math.isfinite(out.item())


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    w, tok = torch.randn(9, 4, device=DEV), torch.tensor([1, 2], device=DEV)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            embedding(tok, fwd.make_dual(w, torch.ones_like(w)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            embedding(tok, fwd.make_dual(w.clone().requires_grad_(True), torch.ones_like(w)))
        assert embedding(tok, w).shape == (2, 4)


def test_forward_mode_through_the_gradient_is_refused():
    import torch.autograd.forward_ad as fwd

    w, tok = torch.randn(9, 4, device=DEV, requires_grad=True), torch.tensor([1, 2], device=DEV)
    out = embedding(tok, w)
    with fwd.dual_level():
        g = fwd.make_dual(torch.ones(2, 4, device=DEV), torch.ones(2, 4, device=DEV))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, w, g)
