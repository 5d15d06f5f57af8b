"""AdamW with 8-bit moments by its definition, in 64 bits on the CPU with numpy (test infrastructure only)."""
from __future__ import annotations

import math

import numpy as np

BLOCK = 64


def random_bits(ids, seed):
    with np.errstate(over="ignore"):
        h = (np.asarray(ids, dtype=np.uint64).astype(np.uint32) * np.uint32(0x9E3779B1)) ^ np.uint32(seed & 0xFFFFFFFF)
        h = (h ^ (h >> np.uint32(16))) * np.uint32(0x85EBCA6B)
        h = (h ^ (h >> np.uint32(13))) * np.uint32(0xC2B2AE35)
        return h ^ (h >> np.uint32(16))


def grid():
    """The 120 e4m3 magnitudes up to 480 (448 is the largest the format holds; nothing here goes beyond 256)."""
    return np.array([i * 2.0**-9 for i in range(8)] + [2.0**e * (1 + f / 8) for e in range(-6, 9) for f in range(8)])


def block_scales(x):
    """The power of two of each 64 elements: the largest magnitude lies in [128, 256) of them; NaN where it is not finite
    or beyond fp32, 1 where all are zero."""
    pad = np.concatenate([np.abs(x), np.zeros(-len(x) % BLOCK)]).reshape(-1, BLOCK)
    out = []
    for row in pad:
        top = row.max()       # NaN stays NaN
        if top == 0:
            out.append(1.0)
        elif not top < 2.0**128:
            out.append(math.nan)
        else:
            out.append(2.0 ** max(math.frexp(top)[1] - 8, -126))
    return np.array(out)


def store(x, u, positive):
    """x rounded stochastically to code * scale -> (values of the codes, scales)."""
    scale = block_scales(x)
    each = np.repeat(scale, BLOCK)[: len(x)]
    g = grid()
    ok = ~np.isnan(each)
    y = np.where(ok, np.abs(x) / np.where(ok, each, 1.0), 0.0)
    lower = np.searchsorted(g, y, side="right") - 1
    step = g[lower + 1] - g[lower]
    up = np.floor((y - g[lower]) / step + u) >= 1
    code = lower + up
    if positive:
        code = np.where((code == 0) & (x > 0), 1, code)
    code = np.where(ok, code, 0)
    if positive:
        code = np.where(~ok & (x > 0), 1, code)
    return np.where((code > 0) & (x < 0), -1.0, 1.0) * g[code], scale


def step(params, grads, ms, vs, m_scales, v_scales, k, lr, betas, eps, decay, seed=0, max_norm=0.0, first=0, sumsq=None):
    """Lists of 1-d float64 arrays (moments as values of codes where scales are given) -> the same lists after the step,
    with the unrounded updates' sizes for error bounds."""
    b1, b2 = betas
    coef = 1.0
    if max_norm > 0:
        total = sum(float((g * g).sum()) for g in grads) if sumsq is None else sumsq
        c = max_norm / (math.sqrt(total) + 1e-6) if not math.isnan(total) else math.nan
        coef = c if c < 1 or math.isnan(c) else 1.0
    key = int(random_bits([k], seed)[0])
    out = []
    with np.errstate(all="ignore"):
        for i, (p, g, m, v) in enumerate(zip(params, grads, ms, vs)):
            if m_scales[i] is not None:
                m = m * np.repeat(m_scales[i], BLOCK)[: len(p)]
                v = v * np.repeat(v_scales[i], BLOCK)[: len(p)]
            g = g * coef
            m = b1 * m + (1.0 - b1) * g
            v = b2 * v + (1.0 - b2) * (g * g)
            mf, vf = m.astype(np.float32).astype(np.float64), v.astype(np.float32).astype(np.float64)
            move = lr / (1 - b1**k) * (mf / (np.sqrt(vf) / math.sqrt(1 - b2**k) + eps))
            q = p * (1 - lr * decay) - move
            if m_scales[i] is None:
                out.append((q, mf, vf, None, None, move))
                continue
            r = random_bits(np.arange(len(p), dtype=np.uint64), int(random_bits([first + i], key)[0]))
            um, uv = (r & np.uint32(0xFFFF)) / 65536.0, (r >> np.uint32(16)) / 65536.0
            mc, a = store(m, um, False)
            vc, b = store(v, uv, True)
            out.append((q, mc, vc, a, b, move))
    return out
