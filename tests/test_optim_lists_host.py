"""The rule by which an optimizer step refuses tensors that share memory, against the bytes themselves (no GPU)."""
import random

import pytest
import torch

CODES = torch.float8_e4m3fn


def _bytes(t):
    a = t.data_ptr()
    return a, a + t.numel() * t.element_size()


def _meet(x, y):
    return x[0] < y[1] and y[0] < x[1]


def _expected(lists):
    p, g, m, v, a, b = lists
    flat = [_bytes(t) for x in (p, m, v, a, b) for t in x if t is not None]
    if any(_meet(x, y) for i, x in enumerate(flat) for y in flat[:i]):
        return "two parameters, moments or scales share memory"
    if any(_meet(x, _bytes(t)) for x in flat for t in g):
        return "a gradient shares memory with what the step writes"
    return None


def _lists(r, order, n):
    """An optimizer's tensors cut from one buffer: list by list, tensor by tensor, or in any order, with gaps here and there."""
    sizes = [r.choice([1, 5, 64, 65, 130]) for _ in range(n)]
    wide = [r.random() < 0.5 for _ in range(n)]
    need = []                                                   # (kind, tensor, bytes)
    for i, k in enumerate(sizes):
        need += [(0, i, 4 * k), (1, i, 4 * k)] + [(j, i, k if wide[i] else 4 * k) for j in (2, 3)]
        need += [(j, i, -(-k // 64) * 4) for j in (4, 5)] if wide[i] else []
    if order == "lists":
        kinds = r.sample(range(6), 6)
        need.sort(key=lambda x: (kinds[x[0]], x[1]))
    elif order == "tensors":
        need.sort(key=lambda x: (x[0] > 1, x[1] if x[0] > 1 else x[0], (0, 1, 2, 4, 3, 5)[x[0]]))
    else:
        r.shuffle(need)
    buf, at, place = torch.zeros(8 * 6 * 560 * n, dtype=torch.uint8), 0, {}
    for kind, i, size in need:
        at += 4 * r.choice([0, 0, 0, 1, 7])
        place[kind, i] = [at, size]
        at += -(-size // 4) * 4
    return buf, place, sizes, wide


@pytest.mark.parametrize("order", ["lists", "tensors", "any"])
@pytest.mark.parametrize("seed", range(25))
def test_shared_memory_is_what_the_bytes_say(order, seed):
    from mpnn_amd import _lib

    shared = _lib.host().shared_memory
    r = random.Random(seed)
    for n in (1, 2, 3, 9, 40):
        buf, place, sizes, wide = _lists(r, order, n)

        def tensors():
            out = [[None] * n for _ in range(6)]
            for (kind, i), (at, size) in place.items():
                t = buf[at:at + size]
                out[kind][i] = t.view(CODES) if kind in (2, 3) and wide[i] else t.view(torch.float32)
            return out

        assert shared(*tensors()) is None is _expected(tensors())
        for _ in range(12):                                      # one of them lies elsewhere
            key = r.choice(list(place))
            old = place[key][0]
            other = r.choice(list(place.values()))
            place[key][0] = max(0, other[0] + 4 * r.randint(-3, 3))
            assert shared(*tensors()) == _expected(tensors())
            place[key][0] = old
        same = tensors()
        for i in range(1, n):                                    # parameters may have the same gradient
            if sizes[i] == sizes[0]:
                same[1][i] = same[1][0]
        assert shared(*same) is None
