"""The token operators together with the segment reductions, as one training step uses them: a table
looked up by voxel id, attention among the voxels of a region, the regions' means, and the gradients
clipped.  Every operator is checked on the values and gradients that it met inside the step."""
import pytest
import torch

from torchex_b200 import ScatterData, clip_grad_norm_, embedding, grad_norm, scatter_mean, segment_attention
from tests.test_attention_gpu import _check, _definition
from tests.test_grad_clip_gpu import NORM_TOL, _norm64

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


class _Regions(torch.nn.Module):
    def __init__(self, vocab, heads, dim, classes):
        super().__init__()
        width = heads * dim
        self.heads, self.dim = heads, dim
        self.table = torch.nn.Parameter(0.1 * torch.randn(vocab, width, dtype=torch.bfloat16))
        self.qkv = torch.nn.Linear(width, 3 * width, dtype=torch.bfloat16)
        self.head = torch.nn.Linear(width, classes)

    def forward(self, voxels, data, kept):
        x = embedding(voxels, self.table, scale=4.0, padding_idx=0)
        q, k, v = self.qkv(x).view(-1, 3, self.heads, self.dim).unbind(1)  # strided views
        out = segment_attention(q, k, v, data, causal=False, softcap=10.0)
        pooled = scatter_mean(out.flatten(1), data)
        kept.update(x=x, q=q, k=k, v=v, out=out, pooled=pooled)
        for t in kept.values():
            t.retain_grad()
        return self.head(pooled)


@pytest.mark.parametrize("longest", [24, 300])
def test_training_step(longest):
    torch.manual_seed(longest)
    heads, dim, vocab = 4, 32, 700
    lens = torch.randint(1, longest + 1, (3000 // longest + 3,))
    ids = torch.repeat_interleave(torch.arange(lens.numel()), lens)
    ids = ids[torch.randperm(ids.numel())].to(DEV)
    data = ScatterData(ids, lens.to(DEV))
    voxels = torch.randint(0, vocab, (ids.numel(),), device=DEV)
    target = torch.randint(0, 5, (lens.numel(),), device=DEV)
    model = _Regions(vocab, heads, dim, 5).to(DEV)
    optimizer = torch.optim.SGD(model.parameters(), lr=0.1)
    for step in range(3):
        kept = {}
        loss = torch.nn.functional.cross_entropy(model(voxels, data, kept), target)
        optimizer.zero_grad()
        loss.backward()
        assert loss.isfinite()
        # the table: rows of the gradient that reached the lookup, summed by voxel
        half = 2.0 ** -8
        rows = torch.where((voxels != 0)[:, None], kept["x"].grad.double(), 0.0)
        total = torch.zeros(vocab, heads * dim, dtype=torch.float64, device=DEV).index_add_(0, voxels, rows) * 4
        size = torch.zeros_like(total).index_add_(0, voxels, rows.abs()) * 4
        count = torch.bincount(voxels, minlength=vocab).double()[:, None]
        assert ((model.table.grad.double() - total).abs() <= (half + 2 ** -22) * total.abs() + count * 2 ** -23 * size + 1e-38).all()
        # attention: with the gradient that the mean sent back
        g = kept["out"].grad
        want = _definition(kept["q"].detach(), kept["k"].detach(), kept["v"].detach(), g, ids, lens.numel(), dim ** -0.5, False, 10.0, None)
        _check([kept["out"].detach(), kept["q"].grad, kept["k"].grad, kept["v"].grad], want)
        # the mean's gradient: an even share of the region's, rounded to bf16 on its way into the attention
        share = (kept["pooled"].grad.double() / lens.to(DEV)[:, None].double())[ids].view_as(g)
        assert ((g.double() - share).abs() <= (half + 2 ** -22) * share.abs() + 1e-38).all()
        before = [p.grad.clone() for p in model.parameters()]
        full = _norm64(before)
        norm = clip_grad_norm_(model.parameters(), 0.25 * full)
        assert abs(norm.item() - full) <= NORM_TOL * full
        after = grad_norm([p.grad for p in model.parameters()]).item()
        assert abs(after - 0.25 * full) <= 0.25 * full * 2 ** -8  # every value rounded by at most half a step
        optimizer.step()
