"""Attention within segments on fp16 values whose probabilities or gradients of scores are far below fp16's smallest
normal number, 2^-14, although the results are not.

The bounds are those of test_attention_gpu, but for what rounding of tiny values may cost.  P and dS are multiplied by a
power of two before they are rounded to fp16, whose values are at least 2^-24 apart, so that
  * a P is off by at most 2^-25 / 2^7 in the forward pass (P is relative to a maximum that may be 2^8 too small, and
    2^8 2^7 = 2^15 is then the largest), and 2^-25 / 2^15 in the backward pass, where P is at most 1;
  * a dS is off by at most 2^-25 / 2^f, with 2^f the largest power that keeps 2^f B below 2^15, or 1 if that is larger.
    B = 2 |scale| |g| |v|, the largest of the segment, bounds |dS|; so 2^f >= 2^14 / B.
"""
import pytest
import torch

from tests.test_attention_gpu import DEV, _plan
from torchex_b200 import segment_attention

pytestmark = pytest.mark.gpu

H = 2 ** -11  # half a step of fp16, relative
STEP = 2 ** -25  # half of the smallest step


def _definition(q, k, v, g, lens, causal, scale):
    """Rows in segment order, one query head per key head: [(value, bound)] for o, gq, gk, gv."""
    q, k, v, g = (x.double() for x in (q, k, v, g))
    dim = q.shape[2]
    found = [[torch.zeros_like(x), torch.zeros_like(x)] for x in (q, q, k, v)]
    begin = 0
    for n in lens:
        rows = slice(begin, begin + n)
        begin += n
        qs, ks, vs, gs = (x[rows].transpose(0, 1) for x in (q, k, v, g))
        x = qs @ ks.mT * scale
        d_score = (dim + 4) * 2 ** -24 * (qs.abs() @ ks.abs().mT) * abs(scale) + 2 ** -22 * (x.abs() + 15)
        at = torch.arange(n, device=DEV)
        seen = (at <= at[:, None]) if causal else torch.ones(n, n, dtype=torch.bool, device=DEV)
        x = x.masked_fill(~seen, float("-inf"))
        d_score = torch.where(seen, d_score, 0.0)
        p = torch.softmax(x, -1)
        e = torch.expm1(2 * (d_score + (p * d_score).sum(-1, keepdim=True) + (n + 16) * 2 ** -24))
        o = p @ vs
        sums = (n + 4) * 2 ** -24
        bound_o = H * o.abs() + (p * (H + e) + STEP * 2 ** -7 * seen) @ vs.abs() + STEP
        dp, delta = gs @ vs.mT, (gs * o).sum(-1, keepdim=True)
        d_dp = (dim + 2) * 2 ** -24 * (gs.abs() @ vs.abs().mT)
        # delta is formed from the output and what rounding took from it: two fp16 values, the second off by half a step
        d_delta = (gs.abs() * (bound_o - H * o.abs() + H * H * o.abs())).sum(-1, keepdim=True) \
            + (dim + 2) * 2 ** -24 * (gs * o).abs().sum(-1, keepdim=True)
        ds = p * (dp - delta) * scale
        largest = 2 * abs(scale) * gs.norm(dim=-1).amax(-1) * vs.norm(dim=-1).amax(-1)
        lost = STEP * (largest * 2 ** -14).clamp(max=1.0)[:, None, None] * seen
        d_ds = p * (d_dp + d_delta) * abs(scale) * (1 + e) + (e + H + 2 ** -22) * ds.abs() + lost
        d_p = p * (H + e) + STEP * 2 ** -15 * seen
        terms = [(o, bound_o),
                 (ds @ ks, d_ds @ ks.abs() + sums * (ds.abs() @ ks.abs())),
                 (ds.mT @ qs, d_ds.mT @ qs.abs() + sums * (ds.abs().mT @ qs.abs())),
                 (p.mT @ gs, d_p.mT @ gs.abs() + sums * (p.mT @ gs.abs()))]
        for i, (value, bound) in enumerate(terms):
            if i >= 1:
                bound = bound + H * value.abs() + STEP
            found[i][0][rows], found[i][1][rows] = value.transpose(0, 1), bound.transpose(0, 1)
    return found


def _check(got, want, names=("out", "g_q", "g_k", "g_v")):
    for name, y, (value, bound) in zip(names, got, want):
        worst = float(((y.double() - value).abs() / bound).nan_to_num(9e9).max())
        assert worst <= 1.0, f"{name}: {worst:.3g} of the bound"


def _peaked(n, heads, dim, below):
    """Key 0 takes all the weight but 2^-below of it per other key, and has a value and a gradient of zero; the others'
    values and gradients are positive, so that what they add up to does not cancel."""
    gen = torch.Generator(device=DEV).manual_seed(n + dim)
    q, k, v, g = ((torch.rand(n, heads, dim, generator=gen, device=DEV) + 0.5) for _ in range(4))
    q, k = (q - 1) / 4, (k - 1) / 4
    q[..., 0], k[..., 0], k[0] = 8.0, 0.0, 0.0
    k[0, :, 0] = below * 0.6931 / 8
    v[0], g[0] = 0.0, 0.0
    return [x.half() for x in (q, k, v, g)]


SHAPES = [([600], 16), ([50], 32), ([64, 900], 64), ([500], 128)]  # general kernels, and those for long segments


@pytest.mark.parametrize("lens,dim", SHAPES)
@pytest.mark.parametrize("below", [18, 26])
def test_small_probabilities_reach_the_output(lens, dim, below):
    ids, data = _plan(lens, False)
    parts = [_peaked(n, 2, dim, below) for n in lens]
    q, k, v, g = (torch.cat(x) for x in zip(*parts))
    want = _definition(q, k, v, g, lens, False, 1.0)
    assert want[0][0].abs().max() > 2 ** -22
    _check([segment_attention(q, k, v, data, scale=1.0)], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,dim", [(300, 16), (20, 64), (300, 64), (300, 128)])
@pytest.mark.parametrize("power", [10, 20, 24, 28, 32, 60])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(dtype, n, dim, power, sign):
    """One key is so far above the others that it takes all the weight: the output is its value, off by the roundings of
    the weight and of the output."""
    gen = torch.Generator(device=DEV).manual_seed(power)
    q, k, v = (torch.zeros(n, 1, dim, device=DEV, dtype=dtype) for _ in range(3))
    q[:, 0, 0] = 2.0 ** 15 * (1 + torch.rand(n, generator=gen, device=DEV) / 2).to(dtype)
    k[:, 0, 0] = sign * (800 + 100 * torch.rand(n, generator=gen, device=DEV)).to(dtype)
    k[n // 3, 0, 0] = 1100.0 if sign > 0 else -600.0
    v[:, 0] = (torch.rand(n, dim, generator=gen, device=DEV) + 1).to(dtype)
    ids, data = _plan([n], False)
    out = segment_attention(q, k, v, data, scale=2.0 ** (power - 25))
    want = v[n // 3].double()
    assert ((out.double() - want).abs() <= (torch.finfo(dtype).eps + 2 ** -20) * want).all()
