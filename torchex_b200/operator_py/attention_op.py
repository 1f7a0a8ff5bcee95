"""Softmax attention within the segments of a ``ScatterData``.

A sparse point transformer attends among the voxels of a region, and a language model among the
tokens of a document packed with others into one batch; both are a pooling over the rows of a
segment whose weights depend on the row.  The rows stay where they are, in any order: the plan that
``scatter_sum`` and its like use says which belong together.  The reference has no counterpart.
"""
from __future__ import annotations

import torch

from .. import scatter_ext as _ext


def segment_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, data, scale=None, causal: bool = False,
                      softcap: float = 0.0, slopes=None) -> torch.Tensor:
    """Attention of every row over the rows of its own segment.

    q: [num_total, heads, dim]; k, v: [num_total, kv_heads, dim]; bfloat16 or float16, ``dim`` a
    multiple of 8 up to 128, ``heads`` a multiple of ``kv_heads`` (consecutive query heads share a
    key / value head).  data: ``ScatterData`` of the same num_total.  Returns [num_total, heads, dim].

    scale: factor of the scores, ``dim ** -0.5`` if None; causal: a row sees the rows of its
    segment up to itself, in increasing row order; softcap: scores become
    ``softcap * tanh(score / softcap)`` where it is positive; slopes: float32 [heads], lowers a score
    by ``slopes[head] * distance``, the distance counted in rows of the segment.

    Differentiable once, by q, k and v.  Statistics and sums are fp32; probabilities and
    gradients of scores are rounded to the dtype of q before they are multiplied (float16: after a
    power of two has brought them into its range, so that small gradients keep their bits).  Results
    are bit-reproducible.  Rows that a query does not see have no influence on its results, whatever
    they hold, but for last bits: beside rows that are not finite tiles are added up in another
    (slower) way, and the powers of two of float16 gradients go by the largest rows of the whole
    segment.  A call that records a gradient keeps, beside q, k, v and the output, what rounding took
    from the output, a tensor of the same size."""
    if data._pending is not None:
        data._poll()
    if not isinstance(q, torch.Tensor) or q.ndim != 3:
        raise RuntimeError("q must be [num_total, heads, dim]")
    return _ext.segment_attention(data._plan, q, k, v, q.shape[2] ** -0.5 if scale is None else float(scale), bool(causal),
                                  float(softcap), slopes)
