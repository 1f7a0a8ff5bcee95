"""Refusals of gradient clipping that need no GPU."""
import ctypes

import pytest
import torch

from torchex_b200 import _native, clip_grad_norm_, clip_grads, grad_norm


def _arrays(ptrs, sizes, types):
    n = len(ptrs)
    return (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*sizes), (ctypes.c_int * n)(*types)


def test_c_abi_rejects_bad_arguments():
    lib = _native.lib()
    need = lib.texb_grad_norm_workspace_bytes(2)
    assert need > 0 and lib.texb_grad_norm_workspace_bytes(-1) == 0
    assert lib.texb_grad_norm_workspace_bytes(100_000) > lib.texb_grad_norm_workspace_bytes(1000)

    def norm(ptrs=(256, 512), sizes=(3, 4), types=(0, 1), out=256, ws=256, nbytes=need, count=2):
        p, s, t = _arrays(ptrs, sizes, types)
        return lib.texb_grad_norm(count, p, s, t, out, ws, nbytes, None)

    assert norm(count=-1) == 1
    assert norm(out=None) == 1
    assert norm(sizes=(3, -4)) == 1 and "negative size" in _native.last_error()
    assert norm(types=(0, 9)) == 1 and "dtype" in _native.last_error()
    assert norm(ptrs=(256, None)) == 1
    assert norm(sizes=(1 << 46, 4)) == 2
    assert norm(ws=None) == 3 and norm(nbytes=need - 1) == 3 and norm(ws=252) == 3
    assert lib.texb_grad_norm(2, None, None, None, 256, 256, need, None) == 1

    def clip(outs=(256, 512), types=(0, 1), out_types=(0, 1), max_norm=1.0):
        p, s, t = _arrays((256, 512), (3, 4), types)
        o, _, ot = _arrays(outs, (0, 0), out_types)
        return lib.texb_clip_grads(2, p, s, t, o, ot, max_norm, 256, None, 0, None)

    assert clip(max_norm=-1.0) == 1 and clip(max_norm=float("nan")) == 1
    assert clip(outs=(256, None)) == 1
    assert clip(out_types=(1, 1)) == 2 and "dtype" in _native.last_error()
    assert clip(out_types=(0, 0)) == 1 and "in place" in _native.last_error()
    assert clip() == 3  # all fine but for the workspace


def test_operators_reject_bad_arguments():
    x = torch.ones(3)
    for call in (lambda: grad_norm([x]), lambda: clip_grads([x], 1.0)):
        with pytest.raises(RuntimeError, match="CUDAtensor"):
            call()
    with pytest.raises(RuntimeError, match="at least one"):
        grad_norm([])
    with pytest.raises(RuntimeError, match="at least one"):
        clip_grads([], 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grads([x], bad)
    assert clip_grad_norm_([torch.nn.Parameter(x)], 1.0).item() == 0.0  # no gradient anywhere


def test_forward_mode_is_refused():
    """A norm or a clipped tensor without its derivative would be taken for a constant."""
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        dual = fwd.make_dual(torch.ones(3), torch.ones(3))
        for call in (lambda: grad_norm([dual]), lambda: clip_grads([dual], 1.0), lambda: clip_grads([dual], 1.0, out=[torch.ones(3)])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
