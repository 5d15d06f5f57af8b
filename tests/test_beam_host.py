"""beam_select / beam_reorder without a GPU: refusals, the plan of layouts, and the oracle against brute force."""
import ctypes
import itertools
import math

import pytest
import torch


def test_cpu_tensors_are_refused():
    import mpnn_amd

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mpnn_amd.beam_select(torch.zeros(1, 2, 3), torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mpnn_amd.beam_reorder(torch.zeros(1, 2, 3), torch.zeros(1, 2, dtype=torch.int64))


def test_bad_arguments_are_refused_by_the_library():
    from mpnn_amd import _lib

    lib = _lib.load()
    P = ctypes.c_void_p(4096)

    def select(dtype=0, B=1, W=4, V=21, n=4, logits=P, ws=None, size=0):
        return lib.mpnn_beam_select(logits, dtype, W * V, V, P, None, 0, 0, None, B, W, V, n, P, P, P, ws, size, None)

    for kw in (dict(logits=None), dict(dtype=3), dict(B=0), dict(W=0), dict(W=257), dict(V=0), dict(V=(1 << 22) + 1), dict(n=0),
               dict(n=257), dict(V=100000), dict(V=100000, ws=P, size=64), dict(V=100000, ws=ctypes.c_void_p(4104), size=1 << 30),
               dict(B=1 << 26), dict(B=1 << 24, W=64), dict(B=1 << 20, W=8, V=9000, ws=P, size=1 << 60)):
        assert select(**kw) == -1 and b"mpnn_beam_select" in lib.mpnn_last_error(), kw
    assert lib.mpnn_beam_select_workspace(0, 4, 4, 21, 4) == 0
    assert lib.mpnn_beam_select_workspace(0, 4, 4, 100000, 4) > 0
    assert lib.mpnn_beam_select_workspace(0, 4, 4, 100000, 300) == -1

    def reorder(n=1, B=1, W=2, parent=P, length_all=-1, rank=None, **kw):
        s = dict(data=4096, stride_group=64, stride_beam=32, stride_mid=0, run=32, n_mid=1)
        s.update(kw)
        return lib.mpnn_beam_reorder(n, (_lib.BeamState * 1)(_lib.BeamState(**s)), parent, B, W, length_all, None, rank, None)

    for kw in (dict(n=0), dict(B=0), dict(B=70000), dict(W=0), dict(W=257), dict(parent=None), dict(rank=P), dict(data=None),
               dict(stride_beam=0), dict(B=2, stride_group=0), dict(n_mid=3), dict(run=0), dict(run=1 << 41), dict(run=(1 << 32) + 1, stride_beam=1 << 33), dict(n_mid=0)):
        assert reorder(**kw) == -1 and b"mpnn_beam_reorder" in lib.mpnn_last_error(), kw


def test_layouts():
    from mpnn_amd import _lib

    layout, span = _lib.host().state_layout, _lib.host().state_span
    x = torch.zeros(2, 3, 4, 6, 8)
    assert layout(x, False) == (1, 0, 192) and layout(x, True) == (4, 48, 48)
    assert layout(x[:, :, :, :5], False) == (4, 48, 40) and layout(x[:, :, :, :5], True) == (4, 48, 40)
    assert layout(x[..., 0], False) == (24, 8, 1) and layout(x[..., 0], True) is None
    assert layout(x[..., :7], False) == (24, 8, 7) and layout(x[:, :, :3, :5, :7], False) is None
    assert layout(x[:, :, :1, :1, :1], False) == (1, 0, 1) and layout(x[:, :, :1, 0], True) == (1, 48, 8)
    assert layout(torch.zeros(2, 3), False) == (1, 0, 1) and layout(torch.zeros(2, 3, 5), True) == (5, 1, 1)
    assert span(x) == x.numel() and span(x.expand(2, 3, 4, 6, 8)[:, :, :2]) == 1152 - 96
    assert span(torch.zeros(2, 1, 4).expand(2, 3, 4)) is None
    assert span(torch.zeros(30).as_strided((2, 3, 4), (12, 3, 1))) is None


def test_oracle_finds_the_best_sequences():
    """A search whose beams hold every hypothesis is exhaustive: its ranking equals brute force over all sequences."""
    from oracle import beam_oracle as orc

    V, steps = 3, 3
    tables = torch.randn(V, V, generator=torch.Generator().manual_seed(0)).double()
    lp = torch.log_softmax(tables, -1)
    W = V ** (steps - 1)
    seq = torch.zeros(1, W, steps, dtype=torch.int64)
    scores = torch.full((1, W), -math.inf, dtype=torch.float64)
    scores[0, 0] = 0
    for t in range(steps):
        last = seq[:, :, t - 1] if t else torch.zeros(1, W, dtype=torch.int64)
        scores, parent, token = orc.select(tables[last], scores)
        seq = orc.reorder(seq, parent)
        seq[:, :, t] = token
    every = {s: float(lp[0, s[0]] + sum(lp[s[i - 1], s[i]] for i in range(1, steps))) for s in itertools.product(range(V), repeat=steps)}
    best = sorted(every, key=lambda s: -every[s])[:W]
    assert [tuple(s) for s in seq[0].tolist()] == best
    assert torch.allclose(scores[0], torch.tensor([every[s] for s in best], dtype=torch.float64))
