"""Beam search's two operators on the HIP library: the choice of the next hypotheses and the states that follow it.

`beam_select` ranks all beams x tokens of each group from the model's logits; `beam_reorder` moves the decoder's state
tensors to the chosen parents, in place.  `ProteinMPNN.beam_search` runs on both; they take any decoder's tensors (any
vocabulary up to 2^22 tokens, caches of any layout whose rows are regular).  Neither has a counterpart in the reference.
Inputs must be on a ROCm device (no CPU fallback); nothing here is differentiable, nothing synchronises with the host.

    scores, parent, token = beam_select(logits, scores, bias=mask, forced=finished)     # [B, W] each
    beam_reorder([keys, values], parent, length=decoded)                                # in place
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import call, ptr, stream_ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INT = (torch.int32, torch.int64)


def _on_gpu(t, name, what, dev=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"mpnn_amd.{what}: {name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"mpnn_amd.{what}: `{name}` must be on a ROCm device (got {t.device}); the HIP path has no CPU "
                           "fallback")
    if dev is not None and t.device != dev:
        raise RuntimeError(f"mpnn_amd.{what}: `{name}` is on {t.device}, the other tensors on {dev}")


def _rows(t):
    """t with adjacent elements along its last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def beam_select(logits, scores, bias=None, forced=None, n_out=None):
    """One step of beam search: logits [B, W, V] (fp32, bf16 or fp16, any strides) of W beams in each of B groups, scores
    [B, W] fp32 -> (scores [B, n_out] fp32, parent [B, n_out] int64, token [B, n_out] int64), best first.

    A candidate's score is scores[b, w] + log_softmax(logits[b, w] + bias[b, w])[v], computed in 64 bits and rounded once;
    ties go to the lowest beam, then the lowest token.  bias: fp32, broadcast to [B, W, V]; -inf takes a token out,
    whatever its logit holds.  forced: integers broadcast to [B, W] ([B] counts for all beams of a group); a beam with
    forced >= 0 offers that token alone, at its own score (a finished hypothesis, a position whose token is given).
    n_out: hypotheses kept, W by default, at most 256.  A slot that no candidate is left for has the score -inf and keeps
    its beam (parent = slot % W).  NaN or +inf in a beam's logits or score: one candidate, token 0, score NaN, ranked first."""
    what = "beam_select"
    _on_gpu(logits, "logits", what)
    dev = logits.device
    _on_gpu(scores, "scores", what, dev)
    if logits.dim() != 3 or logits.dtype not in _DTYPES:
        raise ValueError("mpnn_amd.beam_select: logits must be [B, W, V] in fp32, bf16 or fp16")
    B, W, V = logits.shape
    if tuple(scores.shape) != (B, W) or scores.dtype != torch.float32:
        raise ValueError(f"mpnn_amd.beam_select: scores must be fp32 [{B}, {W}], got {scores.dtype} {tuple(scores.shape)}")
    n = W if n_out is None else int(n_out)
    if not (1 <= W <= 256 and 1 <= n <= 256 and 1 <= V <= 1 << 22):
        raise ValueError("mpnn_amd.beam_select: 1..256 beams, 1..256 hypotheses kept, 1..2^22 tokens "
                         f"(got {W}, {n}, {V})")
    logits, scores = _rows(logits), scores.contiguous()
    bb = bw = 0
    if bias is not None:
        _on_gpu(bias, "bias", what, dev)
        if bias.dtype != torch.float32:
            raise ValueError("mpnn_amd.beam_select: bias must be fp32")
        if bias.dim() < 1 or bias.shape[-1] != V:
            raise ValueError(f"mpnn_amd.beam_select: bias must end in the {V} tokens")
        bias = _rows(bias).expand(B, W, V)
        bb, bw = bias.stride(0), bias.stride(1)
    if forced is not None:
        _on_gpu(forced, "forced", what, dev)
        if forced.dtype not in _INT:
            raise ValueError("mpnn_amd.beam_select: forced must be integers")
        if forced.dim() == 1:
            forced = forced.unsqueeze(1)
        forced = forced.to(torch.int64).expand(B, W).contiguous()
    out = torch.empty(B, n, device=dev, dtype=torch.float32)
    parent = torch.empty(B, n, device=dev, dtype=torch.int64)
    token = torch.empty(B, n, device=dev, dtype=torch.int64)
    if B == 0:
        return out, parent, token
    dt = _DTYPES[logits.dtype]
    with torch.cuda.device(dev):
        need = _lib.load().mpnn_beam_select_workspace(dt, B, W, V, n)
        ws = torch.empty(need, device=dev, dtype=torch.uint8) if need > 0 else None
        call("mpnn_beam_select", logits.data_ptr(), dt, logits.stride(0), logits.stride(1), ptr(scores),
             None if bias is None else bias.data_ptr(), bb, bw, ptr(forced), B, W, V, n, ptr(out), ptr(parent), ptr(token),
             ptr(ws), max(need, 0), stream_ptr())
    return out, parent, token


def _layout(x, by_position):
    """(n_mid, stride_mid, run) of a state's dimensions behind [B, W], in elements; None if they are not regular."""
    dims = [(n, s) for n, s in zip(x.shape[2:], x.stride()[2:])]
    head = [dims.pop(0)] if by_position else []
    merged = []
    for n, s in dims:
        if n == 1:
            continue
        if merged and merged[-1][1] == n * s:
            merged[-1] = (merged[-1][0] * n, s)
        else:
            merged.append((n, s))
    run = merged.pop()[0] if merged and merged[-1][1] == 1 else 1
    mid = head + merged
    if len(mid) > 1:
        return None
    n_mid, stride = mid[0] if mid else (1, 0)
    return n_mid, stride, run


def _span(x):
    """Elements from the first to behind the last; None if two indices share one."""
    extent = 1
    for s, n in sorted((s, n) for n, s in zip(x.shape, x.stride()) if n > 1):
        if s < extent:
            return None
        extent += s * (n - 1)
    return extent


def _apart(a, b):
    """Two layouts (start, end, strides, run; bytes) share no byte though their ranges meet: rows of one lie between those
    of the other."""
    strides = [s for s in a[2] + b[2] if s]
    m = min(strides, default=0)
    if not m or any(s % m for s in strides):
        return False
    d = (b[0] - a[0]) % m
    return d >= a[3] and d + b[3] <= m


def beam_reorder(states, parent, length=None, rank=None):
    """states[i][b, j] <- states[i][b, parent[b, j]] for a tensor or a list of them, in place; returns `states`.

    states: [B, W, ...] of any type, e.g. caches; the dimensions behind the beams must be one contiguous run, or one strided
    dimension of such runs (a [B, W, heads, :t, D] prefix is).  parent: integers [B, W]; a parent outside [0, W) leaves its
    row as it is.  length: an int, or integers [B]: only the positions p < length[b] of dimension 2 move, the others are not
    touched.  rank: integers [B, L], with `length`: position p moves where rank[b, p] < length[b] (a decoding order other
    than left to right).  At most 256 beams.  No two states may share memory."""
    what = "beam_reorder"
    seq = [states] if isinstance(states, torch.Tensor) else list(states)
    _on_gpu(parent, "parent", what)
    dev = parent.device
    if parent.dim() != 2 or parent.dtype not in _INT:
        raise ValueError("mpnn_amd.beam_reorder: parent must be integers [B, W]")
    B, W = parent.shape
    if not 1 <= W <= 256 or B > 65535:
        raise ValueError(f"mpnn_amd.beam_reorder: 1..256 beams and at most 65535 groups (got {W}, {B})")
    if rank is not None and length is None:
        raise ValueError("mpnn_amd.beam_reorder: rank needs a length")
    L = None
    table, spans = [], []
    for x in seq:
        _on_gpu(x, "states", what, dev)
        if x.dim() < 2 or x.shape[0] != B or x.shape[1] != W:
            raise ValueError(f"mpnn_amd.beam_reorder: a state must be [{B}, {W}, ...], got {tuple(x.shape)}")
        if x.requires_grad:
            raise RuntimeError("mpnn_amd.beam_reorder moves states in place: they may not require gradients")
        if length is not None:
            if x.dim() < 3 or L not in (None, x.shape[2]):
                raise ValueError("mpnn_amd.beam_reorder: with a length, every state must be [B, W, positions, ...]")
            L = x.shape[2]
        if x.numel() == 0:
            continue
        lay, extent, item = _layout(x, length is not None), _span(x), x.element_size()
        if lay is None:
            raise ValueError("mpnn_amd.beam_reorder: a state's rows must be contiguous, or one strided dimension of "
                             f"contiguous runs (got strides {x.stride()} of {tuple(x.shape)})")
        if extent is None:
            raise ValueError("mpnn_amd.beam_reorder: rows of a state share memory")
        sb, sw = (x.stride(0) if B > 1 else 0) * item, (x.stride(1) if W > 1 else 0) * item
        sm, start = lay[1] * item, x.data_ptr()
        table.append((start, sb, sw, sm, lay[2] * item, lay[0]))
        spans.append((start, start + extent * item, (sb, sw, sm if lay[0] > 1 else 0), lay[2] * item))
    spans.sort()
    for i, a in enumerate(spans):
        for b in spans[i + 1:]:
            if b[0] >= a[1]:
                break
            if not _apart(a, b):
                raise ValueError("mpnn_amd.beam_reorder: two states share memory")
    length_all, lengths = -1, None
    if isinstance(length, torch.Tensor):
        _on_gpu(length, "length", what, dev)
        if tuple(length.shape) != (B,) or length.dtype not in _INT:
            raise ValueError(f"mpnn_amd.beam_reorder: length must be an int or integers [{B}]")
        lengths = length.to(torch.int32).contiguous()
    elif length is not None:
        length_all = max(0, min(int(length), 0x7FFFFFFF))
    if rank is not None:
        _on_gpu(rank, "rank", what, dev)
        if rank.dtype not in _INT or (L is not None and tuple(rank.shape) != (B, L)):
            raise ValueError(f"mpnn_amd.beam_reorder: rank must be integers [{B}, {L}]")
        rank = rank.to(torch.int32).contiguous()
    if not table:
        return states
    parent = parent.to(torch.int64).contiguous()
    with torch.cuda.device(dev):
        call("mpnn_beam_reorder", len(table), (_lib.BeamState * len(table))(*table), ptr(parent), B, W, length_all,
             ptr(lengths), ptr(rank), stream_ptr())
    torch.autograd.graph.increment_version(seq)
    return states
