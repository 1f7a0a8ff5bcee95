"""Refusals of the attention within segments that need no GPU."""
import ctypes

import pytest
import torch

from torchex_b200 import _native, scatter_ext, segment_attention


def _problem(**changes):
    p = _native.AttentionProblem()
    for name in ("q", "k", "v", "sid", "offsets", "out", "lse", "g", "g_q", "g_k", "g_v"):
        setattr(p, name, 4096)
    p.q_strides[:], p.k_strides[:], p.v_strides[:], p.g_strides[:] = (128, 32), (64, 32), (64, 32), (128, 32)
    p.dtype, p.n, p.num_segments, p.max_count, p.heads, p.kv_heads, p.dim, p.scale = 1, 10, 3, -1, 4, 2, 32, 1.0
    for name, value in changes.items():
        if name.endswith("strides"):
            getattr(p, name)[:] = value
        else:
            setattr(p, name, value)
    return ctypes.byref(p)


def test_c_abi_rejects_bad_arguments():
    lib = _native.lib()
    need = lib.texb_attention_workspace_bytes(10, 4, 2, 1)
    assert need > lib.texb_attention_workspace_bytes(10, 4, 2, 0) > 0 and lib.texb_attention_workspace_bytes(-1, 4, 2, 0) == 0
    for call, nbytes in ((lib.texb_attention_forward, lib.texb_attention_workspace_bytes(10, 4, 2, 0)),
                         (lib.texb_attention_backward, need)):
        assert call(None, 4096, nbytes, None) == 1
        for status, changes in [
                (2, dict(dtype=0)), (2, dict(dtype=7)), (1, dict(n=-1)), (2, dict(n=1 << 31)), (1, dict(num_segments=-1)),
                (1, dict(num_segments=0)), (1, dict(heads=0)), (1, dict(kv_heads=0)), (1, dict(kv_heads=3)), (1, dict(dim=0)),
                (2, dict(dim=12)), (2, dict(dim=136)), (1, dict(softcap=-1.0)), (1, dict(softcap=float("nan"))),
                (1, dict(scale=float("nan"))), (1, dict(scale=float("inf"))), (1, dict(softcap=float("inf"))), (1, dict(q=None)), (1, dict(v=None)), (1, dict(sid=None)), (1, dict(offsets=None)),
                (1, dict(out=None)), (2, dict(k=4104)), (2, dict(q_strides=(132, 32))), (2, dict(v_strides=(64, 30))),
                (2, dict(heads=65535, kv_heads=65535))]:
            assert call(_problem(**changes), 4096, nbytes, None) == status, changes
            assert _native.last_error()
        assert call(_problem(), None, 0, None) == 3 and call(_problem(), 4096, nbytes - 1, None) == 3
        assert call(_problem(n=0), None, 0, None) == 0  # nothing to do
    assert lib.texb_attention_backward(_problem(lse=None), 4096, need, None) == 1
    assert lib.texb_attention_backward(_problem(g_k=None), 4096, need, None) == 1  # without g_v


class _NoPlan:
    _pending = None
    _plan = None


def test_operator_rejects_bad_arguments():
    q = torch.zeros(4, 2, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="num_total, heads, dim"):
        segment_attention(q[0], q, q, _NoPlan())
    with pytest.raises(TypeError):
        segment_attention(q, q, q, _NoPlan())
    assert callable(scatter_ext.segment_attention)


def test_c_abi_rejects_caps_out_of_range():
    """A cap whose factors (2 scale / cap, cap, each in units of log2) leave fp32 would turn scores of 0 into NaN."""
    lib = _native.lib()
    need = lib.texb_attention_workspace_bytes(10, 4, 2, 1)
    for changes in (dict(softcap=1e-45), dict(softcap=3e38), dict(softcap=1e-30, scale=1e10)):
        assert lib.texb_attention_forward(_problem(**changes), 4096, need, None) == 2, changes
        assert lib.texb_attention_backward(_problem(**changes), 4096, need, None) == 2, changes
        assert "softcap" in _native.last_error()


def test_c_abi_rejects_scales_out_of_range():
    """A scale whose factor in units of log2 leaves fp32 would turn scores of 0 into NaN."""
    lib = _native.lib()
    need = lib.texb_attention_workspace_bytes(10, 4, 2, 1)
    for scale in (3e38, -3e38):
        for call in (lib.texb_attention_forward, lib.texb_attention_backward):
            assert call(_problem(scale=scale), 4096, need, None) == 2
            assert "scale" in _native.last_error()
