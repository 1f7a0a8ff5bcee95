"""Rows of a table by token, and the gradient of the table.

The lookup is ``gather_back`` for a table of parameters (one row per token or voxel id), and its
gradient is ``scatter_sum`` of the output's gradient with the tokens as segment ids: the tokens
are sorted and each table row receives the sum of its tokens' rows in one pass, without atomics.
The reference has no counterpart; its users call ``torch.nn.functional.embedding``.
"""
from __future__ import annotations

import torch

from .. import scatter_ext as _ext


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx=None) -> torch.Tensor:
    """``scale * weight[tokens]``: ``tokens`` (int32 or int64, any shape), ``weight`` [vocab, dim]
    (float32, bfloat16 or float16) -> ``[*tokens.shape, dim]`` in the dtype of ``weight``, scaled in
    fp32 and rounded once.

    The gradient of ``weight`` is dense (every row written), summed in fp32 and rounded once, and
    bit-reproducible.  Tokens equal to ``padding_idx`` (negative: counted from the end) take no
    part in it.  Neither direction synchronises with the device, so a token outside
    ``[0, vocab)`` cannot raise: its row of the output is zero, it takes no part in the gradient,
    and it is counted (``_native.device_bad_indices()``).  Differentiable once."""
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2:
        raise RuntimeError("weight must be [vocab, dim]")
    pad = -1
    if padding_idx is not None:
        vocab = weight.shape[0]
        if not -vocab <= padding_idx < vocab:
            raise ValueError(f"padding_idx {padding_idx} is outside a table of {vocab} rows")
        pad = int(padding_idx) % vocab
    return _ext.embedding(tokens, weight, float(scale), pad)
