"""8-bit moments without a GPU: refusals, the stored format, conversion, and the oracle's rounding."""
import ctypes
import math

import numpy as np
import pytest
import torch


def test_library_refuses_bad_arguments():
    from mpnn_amd import _lib

    lib = _lib.load()
    one = lambda x=4096: (ctypes.c_void_p * 1)(x)   # noqa: E731
    size = lambda x: (ctypes.c_longlong * 1)(x)     # noqa: E731

    def step(n=1, p=4096, g=4096, a=4096, b=4096, numel=100, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, k=1, first=0):
        return lib.mpnn_adamw_mixed(n, one(p), one(g), one(), one(), one(a), one(b), size(numel), lr, b1, b2, eps, wd, k, 0, first,
                                    None, 0.0, None, None)

    for kw in (dict(n=0), dict(p=None), dict(g=None), dict(a=None), dict(b=None), dict(numel=0), dict(numel=1 << 32), dict(lr=-1.0),
               dict(b1=1.0), dict(b2=1.0), dict(eps=-1.0), dict(wd=-1.0), dict(k=0), dict(first=-1), dict(lr=math.nan)):
        assert step(**kw) == -1 and b"mpnn_adamw_mixed" in lib.mpnn_last_error(), kw
    assert lib.mpnn_grad_sumsq_parts(1, one(), size(0), ctypes.c_void_p(4096), None) == -1
    assert lib.mpnn_grad_sumsq_parts(1, one(), size(5), None, None) == -1
    assert lib.mpnn_grad_sumsq_parts(32769, one(), size(5), ctypes.c_void_p(4096), None) == -1


def test_optimizer_refusals_without_a_gpu():
    from mpnn_amd import training
    from mpnn_amd.optim import AdamW, adamw_step

    p = torch.nn.Parameter(torch.zeros(5000))
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([p], state_bits=16)
    opt = AdamW([p], state_bits=8)
    p.grad = torch.zeros(5000)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        opt.step()
    z = torch.zeros(100)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        adamw_step([z], [z], [z], [z], [None], [None], step=1)
    with pytest.raises(RuntimeError, match="ROCm"):
        training.make_optimizer(torch.nn.Linear(2, 2), state_bits=8)


def test_stored_format_and_conversion():
    from mpnn_amd.optim import pack_moment, unpack_moment

    g = torch.Generator().manual_seed(0)
    x = torch.randn(7, 31, generator=g) * torch.exp(4 * torch.randn(7, 31, generator=g))
    x[2] = 0
    codes, scale = pack_moment(x)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape and scale.shape == (4,)
    low = scale.repeat_interleave(64)[:217].view(7, 31) * 2.0**-10          # half of the lowest code's step
    assert bool(((unpack_moment(codes, scale) - x).abs() <= torch.maximum(x.abs() * 2.0**-4, low)).all())
    again = pack_moment(unpack_moment(codes, scale))
    assert torch.equal(unpack_moment(*again), unpack_moment(codes, scale)), "what is stored converts without loss"
    v = x.abs() ** 2 * 1e-6
    codes, scale = pack_moment(v, positive=True)
    assert bool((unpack_moment(codes, scale)[v > 0] > 0).all()) and bool((unpack_moment(codes, scale)[v == 0] == 0).all())
    x[3, 0] = math.inf
    codes, scale = pack_moment(x)
    assert torch.isnan(scale).tolist() == [False, True, False, False]
    assert pack_moment(torch.zeros(0))[1].numel() == 0


def test_oracle_grid_is_the_format():
    from oracle import adamw_oracle as orc

    every = torch.arange(0x79, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()   # codes up to 256
    np.testing.assert_array_equal(orc.grid()[:0x79], every)


def test_oracle_rounding_is_unbiased_and_reproducible():
    """Over all 65536 draws the mean of the stored value is the value: exactly, to the draws' step of 2^-16."""
    from oracle import adamw_oracle as orc

    u = np.arange(65536) / 65536.0
    for value in (1.0, 0.37, 3e-3, 1.2e-5, 255.9):
        x = np.full(65536, value)
        x[::64] = 200.0                        # the block's scale is 1
        q, scale = orc.store(x, u, False)
        assert (scale == 1.0).all()
        mine = np.arange(65536) % 64 != 0
        assert abs(q[mine].mean() - value) <= 2.0**-9 * max(value, 2.0**-6) / 8 + 2.0**-16 * value
    r = orc.random_bits(np.arange(1 << 16), 7)
    assert len(set(r.tolist())) > 65000 and abs((r & 0xFFFF).mean() / 65536 - 0.5) < 0.01
