"""Beam search on torch CUDA tensors: the selection over beams and vocabulary, and the reordering of what beams carry.

The reference decodes greedily only (llama3.py:320).  Both operators enqueue their kernels on the current stream of the tensors'
device and return, and can be captured into a graph; arguments that do not fit raise ValueError before anything is enqueued.
Neither has a derivative: outside torch.no_grad() they refuse tensors that require a gradient, and tensors with a forward-mode gradient.
"""
from __future__ import annotations

from .paged import _ops


def beam_select(logits, scores, best=None, *, done=None, eos_id=None):
    """The best continuations of every sequence's beams, by scores[b, k] + log softmax(logits[b, k])[v].

    logits  [batch, beams, vocab] fp32, bfloat16 or float16, last dimension contiguous; up to 256 beams
    scores  [batch, beams] fp32: the beams' sums of log probabilities (-inf: no beam)
    best    how many continuations, up to 64; as many as there are beams by default
    done    [batch, beams] bool: beams that ended; such a beam has one continuation, the token eos_id at its own score
    Returns scores [batch, best] fp32 in falling order (equal ones by beam, then token), tokens and parents (beams of the same
    sequence) [batch, best] int32, and done [batch, best] bool: the parent had ended, or the token is eos_id.  A score that is
    -inf, +inf or NaN is no continuation; a place that none is left for has score -inf, the token eos_id (or 0), parent 0, done.
    Beams with the same logits have the same sum of exponentials; of different ones, whose sums are of fp32 terms, scores closer
    than 2^-19 may come in either order.
    """
    return _ops().beam_select(logits, scores, best, done, eos_id)


def beam_reorder(states, parents):
    """In place, row b * beams + j of every state becomes what row b * beams + parents[b, j] was.

    states   a list of tensors [batch * beams, ...] of any type: recurrent states, page tables, token histories, cache rows; a row
             is a contiguous run, or equal runs at equal distances (`cache[:, :, first:last]`);
             no two states may share memory
    parents  [batch, beams] int32, any of a sequence's beams (up to 256), several times too; a number outside leaves its row as it is
    """
    _ops().beam_reorder(states, parents)
