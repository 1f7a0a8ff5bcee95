from .scatter_op import (GetPreSumFunction, ScatterData, ScatterMaxFunction, ScatterMeanFunction,
                         ScatterSumFunction, gather_back, getPreSum, ingroup_inds, ingroup_rank, scatter_max,
                         scatter_mean, scatter_mean_max, scatter_multi, scatter_sum, ScatterMeanMaxFunction)
from .attention_op import segment_attention
from .clip_op import clip_grad_norm_, clip_grads, grad_norm
from .embedding_op import embedding
from .timer import TorchTimer

__all__ = ["TorchTimer", "scatter_sum", "scatter_mean", "scatter_max", "getPreSum", "ScatterData",
           "ScatterSumFunction", "ScatterMeanFunction", "ScatterMaxFunction", "GetPreSumFunction",
           "ingroup_inds", "ingroup_rank", "gather_back", "scatter_mean_max", "scatter_multi", "ScatterMeanMaxFunction",
           "embedding",
           "grad_norm", "clip_grads", "clip_grad_norm_", "segment_attention"]
