"""Beam search's two operators on the HIP library: the choice of the next hypotheses and the states that follow it.

`beam_select` ranks all beams x tokens of each group from the model's logits; `beam_reorder` moves the decoder's state
tensors to the chosen parents, in place.  `ProteinMPNN.beam_search` runs on both; they take any decoder's tensors (any
vocabulary up to 2^22 tokens, caches of any layout whose rows are regular).  Neither has a counterpart in the reference.
Inputs must be on a ROCm device (no CPU fallback); nothing here is differentiable, nothing synchronises with the host.

    scores, parent, token = beam_select(logits, scores, bias=mask, forced=finished)     # [B, W] each
    beam_reorder([keys, values], parent, length=decoded)                                # in place
"""
from __future__ import annotations

from ._lib import host_call


def beam_select(logits, scores, bias=None, forced=None, n_out=None):
    """One step of beam search: logits [B, W, V] (fp32, bf16 or fp16, any strides) of W beams in each of B groups, scores
    [B, W] fp32 -> (scores [B, n_out] fp32, parent [B, n_out] int64, token [B, n_out] int64), best first.

    A candidate's score is scores[b, w] + log_softmax(logits[b, w] + bias[b, w])[v], computed in 64 bits and rounded once;
    ties go to the lowest beam, then the lowest token.  bias: fp32, broadcast to [B, W, V]; -inf takes a token out,
    whatever its logit holds.  forced: integers broadcast to [B, W] ([B] counts for all beams of a group); a beam with
    forced >= 0 offers that token alone, at its own score (a finished hypothesis, a position whose token is given).
    n_out: hypotheses kept, W by default, at most 256.  A slot that no candidate is left for has the score -inf and keeps
    its beam (parent = slot % W).  NaN or +inf in a beam's logits or score: one candidate, token 0, score NaN, ranked first."""
    return host_call("mpnn_beam_select", "beam_select", logits, scores, bias, forced, n_out)


def beam_reorder(states, parent, length=None, rank=None):
    """states[i][b, j] <- states[i][b, parent[b, j]] for a tensor or a list of them, in place; returns `states`.

    states: [B, W, ...] of any type, e.g. caches; the dimensions behind the beams must be one contiguous run, or one strided
    dimension of such runs (a [B, W, heads, :t, D] prefix is).  parent: integers [B, W]; a parent outside [0, W) leaves its
    row as it is.  length: an int, or integers [B]: only the positions p < length[b] of dimension 2 move, the others are not
    touched.  rank: integers [B, L], with `length`: position p moves where rank[b, p] < length[b] (a decoding order other
    than left to right; 64-bit integers compare as such).  At most 256 beams.  No two states may share memory
    (rows of one may lie between the other's: keys and values of one [B, W, 2, heads, T, D] buffer)."""
    return host_call("mpnn_beam_reorder", "beam_reorder", states, parent, length, rank)
