"""Beam search's operators by their definitions, in 64 bits on the CPU (test infrastructure only)."""
from __future__ import annotations

import math

import torch


def select(logits, scores, bias=None, forced=None, n_out=None):
    """-> (scores [B, n] float64, parent, token): every candidate of a group in a list, sorted by (score, beam, token)."""
    B, W, V = logits.shape
    n = W if n_out is None else n_out
    x = logits.double()
    if bias is not None:
        bias = bias.double().expand(B, W, V)
        x = torch.where(bias == -math.inf, bias, x + bias)
    if forced is not None:
        forced = (forced.unsqueeze(1) if forced.dim() == 1 else forced).expand(B, W)
    out = torch.full((B, n), -math.inf, dtype=torch.float64)
    parent = torch.zeros(B, n, dtype=torch.int64)
    token = torch.zeros(B, n, dtype=torch.int64)
    for b in range(B):
        cand = []
        for w in range(W):
            s, row = float(scores[b, w]), x[b, w]
            if forced is not None and int(forced[b, w]) >= 0:
                cand.append((s, w, min(int(forced[b, w]), V - 1)))
                continue
            live = row != -math.inf
            if bool((row[live].isnan() | (row[live] == math.inf)).any()) or math.isnan(s) or s == math.inf:
                cand.append((math.nan, w, 0))
                continue
            lp = (s + (row - torch.logsumexp(row, 0))).tolist()
            cand += [(c, w, v) for v, c in enumerate(lp) if bool(live[v])]
        cand = [c for c in cand if c[0] != -math.inf]
        cand.sort(key=lambda c: (-math.inf if math.isnan(c[0]) else -c[0], not math.isnan(c[0]), c[1], c[2]))
        for j in range(n):
            if j < len(cand):
                out[b, j], parent[b, j], token[b, j] = cand[j]
            else:
                parent[b, j] = j % W
                if forced is not None:
                    token[b, j] = min(max(int(forced[b, j % W]), 0), V - 1)
    return out, parent, token


def select_large(logits, scores, n):
    """select() without bias and forced tokens, for finite inputs and scores of -inf, by a stable sort of whole groups."""
    B, W, V = logits.shape
    x = logits.double()
    c = scores.double()[..., None] + (x - torch.logsumexp(x, -1, keepdim=True))
    s, i = torch.sort(c.view(B, -1), dim=1, descending=True, stable=True)
    s, i = s[:, :n], i[:, :n]
    slot = torch.arange(n).expand(B, n) % W
    dead = s == -math.inf
    return s, torch.where(dead, slot, i // V), torch.where(dead, torch.zeros_like(i), i % V)


def reorder(state, parent, length=None, rank=None):
    """A new tensor: state[b, j] = old state[b, parent[b, j]], at the positions that move."""
    out = state.clone()
    B, W = parent.shape
    for b in range(B):
        for j in range(W):
            p = int(parent[b, j])
            if not 0 <= p < W:
                continue
            if length is None:
                out[b, j] = state[b, p]
                continue
            n = int(length[b]) if isinstance(length, torch.Tensor) else length
            pos = torch.arange(state.shape[2]) if rank is None else rank[b]
            live = pos < n
            out[b, j, live] = state[b, p, live]
    return out
