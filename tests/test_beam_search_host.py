"""Inputs that beam_search refuses (no GPU: the check itself, on tensors of any device)."""
import pytest
import torch


def _inputs(B=2, L=5):
    return dict(mask=torch.ones(B, L), residue_idx=torch.zeros(B, L, dtype=torch.int64),
                chain_encoding_all=torch.ones(B, L, dtype=torch.int64))


def test_inputs_beside_x():
    from mpnn_amd.engine import _require_batch

    X = torch.zeros(2, 5, 4, 3)
    _require_batch("beam_search", X, **_inputs())
    _require_batch("beam_search", X.double().transpose(0, 1).contiguous().transpose(0, 1), **_inputs())
    for name in _inputs():
        for shape in ((2, 4), (1, 5), (5,), (2, 5, 1), ()):
            bad = _inputs()
            bad[name] = torch.zeros(shape)
            with pytest.raises(ValueError, match=name):
                _require_batch("beam_search", X, **bad)
        bad = _inputs()
        bad[name] = torch.zeros(2, 5, device="meta")
        with pytest.raises(RuntimeError, match=name):
            _require_batch("beam_search", X, **bad)
    for shape in ((2, 5, 4), (2, 5, 3, 3), (2, 5, 4, 4), (5, 4, 3), (5, 2, 4, 3), (10, 4, 3)):
        with pytest.raises(ValueError, match="X must be"):
            _require_batch("beam_search", torch.zeros(shape), **_inputs())
