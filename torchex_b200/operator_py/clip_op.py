"""The norm over all gradients of a model, and gradient clipping by it.

One reduction over a list of tensors of any number and sizes, and the scaled tensors, in two
launches.  The reference has no counterpart; its users call
``torch.nn.utils.clip_grad_norm_``.
"""
from __future__ import annotations

import torch

from .. import scatter_ext as _ext


def grad_norm(grads) -> torch.Tensor:
    """2-norm over all values of a sequence of tensors (float32, bfloat16 or float16, dense in
    memory, on one device): a float32 tensor without axes on that device.  Does not synchronise.
    Not differentiable: tensors that require a gradient are taken under ``torch.no_grad()`` only."""
    return _ext.grad_norm(list(grads))


def clip_grads(grads, max_norm: float, out=None):
    """``(clipped, norm)``: every tensor of ``grads`` times ``min(1, max_norm / (norm + 1e-6))`` with
    ``norm = grad_norm(grads)``, rounded once.

    ``out`` (a sequence, one tensor per gradient, of the same shape and strides) receives the
    results: new tensors if it is None, ``grads`` itself for scaling in place, or for instance the
    float32 gradients that an optimizer keeps beside 16-bit ones (each output has the dtype of its
    gradient or float32).  Not differentiable, as ``grad_norm``.  Outputs overlap neither each other nor another gradient.  Does not
    synchronise; an infinite or NaN norm shows in the results as it does in
    ``torch.nn.utils.clip_grad_norm_`` with ``error_if_nonfinite=False``."""
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return _ext.clip_grads(list(grads), float(max_norm), None if out is None else list(out))


def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_(parameters, max_norm)``: scales the ``grad`` of the
    parameters (a tensor or an iterable of tensors; those without one are passed over) in place
    and returns their norm.  A parameter that is listed twice is refused."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    with torch.no_grad():  # gradients of a backward pass with create_graph require one themselves
        return clip_grads(grads, max_norm, out=grads)[1]
