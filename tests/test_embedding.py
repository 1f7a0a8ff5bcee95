"""Refusals of the table lookup that need no GPU."""
import pytest
import torch

from torchex_b200 import _native, embedding, scatter_ext


def test_c_abi_rejects_bad_arguments():
    lib = _native.lib()
    fwd, bwd, size = lib.texb_embedding_forward, lib.texb_embedding_backward, lib.texb_embedding_backward_workspace_bytes
    assert fwd(None, 3, 4, None, 0, 5, 8, 1.0, None, None) == 1 and "id_bytes" in _native.last_error()
    assert fwd(None, 4, 4, None, 7, 5, 8, 1.0, None, None) == 1 and "dtype" in _native.last_error()
    assert fwd(None, 4, -1, None, 0, 5, 8, 1.0, None, None) == 1
    assert fwd(None, 4, 4, None, 0, 5, 0, 1.0, None, None) == 1
    assert fwd(None, 4, 1 << 31, None, 0, 5, 8, 1.0, None, None) == 2
    assert fwd(None, 4, 4, None, 0, 5, 8, 1.0, None, None) == 1      # NULL pointers
    assert fwd(None, 4, 0, None, 0, 5, 8, 1.0, None, None) == 0      # nothing to do
    assert bwd(None, 8, 4, None, 0, 1 << 31, 8, 1.0, -1, None, None, 0, None) == 2
    assert bwd(1, 8, 4, 1, 0, 5, 8, 1.0, -1, 1, None, 0, None) == 3  # no workspace
    assert bwd(1, 8, 4, 1, 0, 5, 8, 1.0, -1, 1, 256, 16, None) == 3 and "workspace" in _native.last_error()
    assert bwd(None, 8, 0, None, 0, 0, 8, 1.0, -1, None, None, 0, None) == 0
    assert size(-1, 5, 8) == 0 and size(1000, 5000, 8) >= 8_000


def test_operator_rejects_bad_arguments():
    tok, w = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4)
    with pytest.raises(RuntimeError, match="CUDAtensor"):
        embedding(tok, w)
    with pytest.raises(RuntimeError, match=r"\[vocab, dim\]"):
        embedding(tok, w[0])
    for pad in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            embedding(tok, w, padding_idx=pad)
    with pytest.raises(RuntimeError, match="CUDAtensor"):
        scatter_ext.embedding_backward(tok, torch.zeros(3, 4), 5, 1.0, -1)
