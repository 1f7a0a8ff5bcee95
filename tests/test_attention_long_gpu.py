"""The attention kernels for long segments on more tiles, layouts and values than test_attention_gpu reaches, by the same
definition and bounds."""
import pytest
import torch

from tests.test_attention_gpu import DEV, TYPES, _check, _definition, _inputs, _plan, _step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shuffled", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (3, 1, 64), (2, 2, 40)])
def test_long_and_short_segments_together(dtype, causal, shuffled, heads, kv_heads, dim):
    """Dozens of tiles of very different lengths, some of many short segments."""
    lens = [2500, 1, 33, 2100, 0, 700, 128, 5] + [1 + 13 * i % 50 for i in range(40)] + [1500, 256]
    ids, data = _plan(lens, shuffled, 1)
    q, k, v, g = _inputs(sum(lens), heads, kv_heads, dim, dtype, 12)
    want = _definition(q, k, v, g, ids, len(lens), dim ** -0.5, causal, 0.0, None)
    _check(_step(q, k, v, g, data, causal=causal), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim", [(4, 64), (2, 128), (3, 72)])
def test_strides_of_rows_in_segment_order(dtype, heads, dim):
    """Slices of a fused projection, heads in front of rows, heads and rows that are all one."""
    lens = [300, 70, 200]
    n = sum(lens)
    ids, data = _plan(lens, False)
    gen = torch.Generator(device=DEV).manual_seed(2)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device=DEV).to(dtype)

    fused, by_head, one, row = rand(n, 4, heads, dim), rand(4, heads, n, dim).transpose(1, 2), rand(n, 1, dim), rand(1, heads, dim)
    for label, (q, k, v, g) in {
            "fused": fused.unbind(1), "by head": by_head.unbind(0),
            "one head": (one.expand(n, heads, dim), fused[:, 1], one.expand(n, heads, dim), one.expand(n, heads, dim)),
            "one row": (fused[:, 0], fused[:, 1], row.expand(n, heads, dim), row.expand(n, heads, dim))}.items():
        want = _definition(q, k, v, g, ids, len(lens), dim ** -0.5, True, 0.0, None)
        _check(_step(q, k, v, g, data, causal=True), want, label=label)


@pytest.mark.parametrize("shuffled", [False, True])
def test_rows_and_heads_beyond_32_bit_offsets(shuffled):
    n, heads, dim, length = 150_000, 112, 128, 50  # 2.15e9 values of q and of its gradients
    gen = torch.Generator(device=DEV).manual_seed(5)
    q, g = (torch.randn(n, heads, dim, generator=gen, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(n, 1, dim, generator=gen, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    segments = n // length
    ids = torch.arange(n, device=DEV) % segments if shuffled else torch.arange(n, device=DEV) // length
    from torchex_b200 import ScatterData
    got = _step(q, k, v, g, ScatterData(ids, torch.full((segments,), length, device=DEV)))
    for s in (0, segments // 2, segments - 1):
        rows = (ids == s).nonzero()[:, 0]
        part = [x[rows] for x in (q, k, v, g)]
        want = _definition(*part, torch.zeros(length, device=DEV), 1, dim ** -0.5, False, 0.0, None)
        _check([x[rows] for x in got], want, label=str(s))
