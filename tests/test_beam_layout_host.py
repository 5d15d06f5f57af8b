"""beam_reorder's rule for states of one buffer, against the bytes themselves (no GPU)."""
import random

import pytest
import torch


def _bytes(x):
    at = torch.arange(x.untyped_storage().nbytes() // x.element_size()).as_strided(x.shape, x.stride(), x.storage_offset())
    first = at.flatten() * x.element_size()
    return {int(b) + i for b in first for i in range(x.element_size())}


def _view(buf, r):
    """A state [B, W, ...] as a program cuts it out of a buffer: some dimensions indexed away, others sliced, beams first or not."""
    x = buf
    while x.dim() > 5 or (x.dim() > 3 and r.random() < 0.5):
        d = r.randrange(2, x.dim())
        x = x.select(d, r.randrange(x.shape[d]))
    for d in range(2, x.dim()):
        if r.random() < 0.5:
            n = x.shape[d]
            a = r.randrange(n)
            x = x.narrow(d, a, r.randint(1, n - a))
        elif r.random() < 0.2:
            x = x[(slice(None),) * d + (slice(r.randrange(2), None, 2),)]
    if x.dim() > 3 and r.random() < 0.2:
        x = x.transpose(2, 3)
    return x


@pytest.mark.parametrize("seed", range(40))
def test_states_apart_is_what_the_bytes_say(seed):
    from mpnn_amd import _lib

    apart = _lib.host().states_apart
    r = random.Random(seed)
    seen = {True: 0, False: 0, None: 0}
    for _ in range(60):
        B, W = r.randint(1, 3), r.randint(1, 3)
        rest = [r.choice([1, 2, 2, 3, 4, 5]) for _ in range(r.randint(1, 4))]
        if r.random() < 0.3:
            buf = torch.zeros([W, B] + rest, dtype=r.choice([torch.float32, torch.int64])).transpose(0, 1)
        else:
            buf = torch.zeros([B, W] + rest, dtype=r.choice([torch.float32, torch.uint8]))
        x, y = _view(buf, r), _view(buf, r)
        by_position = r.random() < 0.3 and min(x.dim(), y.dim()) > 2
        got = apart(x, y, by_position)
        seen[got] += 1
        if got is not None:
            assert got == (not _bytes(x) & _bytes(y)), (buf.shape, buf.stride(), x.shape, x.stride(), x.storage_offset(), y.shape,
                                                        y.stride(), y.storage_offset(), by_position)
            assert apart(y, x, by_position) == got
    assert seen[True] > 3 and seen[False] > 3


def test_states_apart_of_large_caches():
    """Sizes of a real cache, on memory that is never touched."""
    from mpnn_amd import _lib

    apart = _lib.host().states_apart
    x = torch.empty(4, 16, 2, 16, 4096, 128, dtype=torch.uint8)
    k, v = x[:, :, 0, :, :4001], x[:, :, 1, :, :4001]
    assert apart(k, v, False) and apart(k, x[:, :, 1], False) and apart(k, x[:, :, 0, :, 4001:], False)
    assert not apart(k, x[:, :, 0, :, 4000:], False) and not apart(k, x[:, :, 0, 5], False) and not apart(v, v, False)
    assert apart(x[:, :, 0, 0, ::2], x[:, :, 0, 0, 1::2], False), "rows of one between the other's"
    # so irregular that the rule gives up: refused, not taken for apart
    odd = x.as_strided((4, 16, 4000, 3), (1 << 28, 1 << 24, 1009, 1), 500)
    even = x.as_strided((4, 16, 4000, 3), (1 << 28, 1 << 24, 1013, 1), 4000)
    assert apart(odd, odd.as_strided((4, 16, 4000, 3), (1 << 28, 1 << 24, 1009, 1), 503), False)
    assert not apart(odd, even, False)
