"""B200-native segmented scatter reduction with TorchEx's operator API.

Drop-in for the scatter part of ``torchex``: ``ScatterData``, ``scatter_sum``,
``scatter_mean``, ``scatter_max`` (and ``TorchTimer``), backed by hand-written
sm_100a kernels behind a C ABI (``include/texb_scatter.h``).  Beside them: ``embedding``
(rows of a table by token, and its gradient), ``segment_attention`` (attention within the
segments of a ``ScatterData``) and ``grad_norm`` / ``clip_grads`` / ``clip_grad_norm_``.
"""
from .operator_py import (ScatterData, TorchTimer, clip_grad_norm_, clip_grads, embedding, gather_back, getPreSum,
                          grad_norm, ingroup_inds, ingroup_rank, scatter_max, scatter_mean, scatter_mean_max,
                          scatter_multi, scatter_sum, segment_attention)

__all__ = ["ScatterData", "TorchTimer", "getPreSum", "scatter_max", "scatter_mean", "scatter_sum",
           "ingroup_inds", "ingroup_rank", "gather_back", "scatter_mean_max", "scatter_multi",
           "embedding", "grad_norm", "clip_grads", "clip_grad_norm_", "segment_attention"]
