"""Beam search on torch CUDA tensors: the selection over beams and vocabulary, and the reordering of what beams carry.

The reference decodes greedily only (llama3.py:320).  Both operators enqueue their kernels on the current stream of the tensors'
device and return, and can be captured into a graph; arguments that do not fit raise ValueError before anything is enqueued.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _cabi
from .paged import _KIND, _filled, _form, _ints, _need, _one_device, _planned, _rows, _stream, _tensor

MOST_BEAMS, MOST_BEST = 256, 64
_select_plans: dict = {}
_reorder_plans: dict = {}


def _plan_select(logits, scores, best, done, eos_id):
    _tensor(logits, "logits", 3, tuple(_KIND))
    batch, beams, vocab = logits.shape
    best = beams if best is None else int(best)
    _need(1 <= beams <= MOST_BEAMS, "%d beams: 1 to %d are supported", beams, MOST_BEAMS)
    _need(1 <= best <= MOST_BEST, "best %d: 1 to %d are supported", best, MOST_BEST)
    _need(1 <= vocab < 1 << 24 and batch * beams <= 65535, "logits of shape %s are too large", tuple(logits.shape))
    _need(vocab == 1 or logits.stride(2) == 1, "logits: the last dimension must be contiguous")
    _tensor(scores, "scores", 2, (torch.float32,))
    _need(tuple(scores.shape) == (batch, beams) and scores.is_contiguous(), "scores must be contiguous, %s, got %s", (batch, beams),
          tuple(scores.shape))
    eos = -1 if eos_id is None else int(eos_id)
    _need(eos < vocab and (eos >= 0 or eos_id is None), "eos_id %s is not in the vocabulary of %d", eos_id, vocab)
    if done is not None:
        _tensor(done, "done", 2, (torch.bool, torch.uint8))
        _need(tuple(done.shape) == (batch, beams) and done.is_contiguous(), "done must be contiguous, %s, got %s", (batch, beams),
              tuple(done.shape))
        _need(eos >= 0, "finished beams need an eos_id")
    device = _one_device((("logits", logits), ("scores", scores), ("done", done)))
    sizes = (device.index, batch, beams, vocab, best)
    n = C.c_int64()
    if batch:
        _cabi.check(_cabi.lib().l3_beam_select_workspace(*sizes, C.byref(n)))
    room = -(-n.value // 4)
    arg = _cabi.L3BeamSelect(*sizes, eos, _KIND[logits.dtype], 0, None, None, logits.stride(0) if batch > 1 else 0,
                             logits.stride(1) if beams > 1 else 0, None, None, None, None, None, None, None, room * 4)
    return bytes(arg), device.index, room, (batch, best)


def beam_select(logits, scores, best=None, *, done=None, eos_id=None):
    """The best continuations of every sequence's beams, by scores[b, k] + log softmax(logits[b, k])[v].

    logits  [batch, beams, vocab] fp32, bfloat16 or float16, last dimension contiguous
    scores  [batch, beams] fp32: the beams' sums of log probabilities (-inf: no beam)
    best    how many continuations, up to 64; as many as there are beams by default
    done    [batch, beams] bool: beams that ended; such a beam has one continuation, the token eos_id at its own score
    Returns scores [batch, best] fp32 in falling order (equal ones by beam, then token), tokens and parents (beams of the same
    sequence) [batch, best] int32, and done [batch, best] bool: the parent had ended, or the token is eos_id.  A score that is
    -inf, +inf or NaN is no continuation; a place that none is left for has score -inf, the token eos_id (or 0), parent 0, done.
    """
    try:
        key = (_form(logits), _form(scores), best, _form(done), eos_id)
    except (AttributeError, RuntimeError):
        key = None                                     # not tensors, or not strided ones: refused below
    args = (logits, scores, best, done, eos_id)
    fixed, index, room, shape = _plan_select(*args) if key is None else _planned(_select_plans, key, _plan_select, *args)
    values = scores.new_empty(shape)
    tokens = torch.empty_like(values, dtype=torch.int32)
    parents, over = torch.empty_like(tokens), torch.empty_like(tokens, dtype=torch.bool)
    if shape[0]:
        ws = scores.new_empty(room)                    # of this call: a captured graph has one of its own
        arg = _cabi.L3BeamSelect.from_buffer_copy(fixed)
        arg.stream, arg.logits, arg.scores, arg.workspace = _stream(index), logits.data_ptr(), scores.data_ptr(), ws.data_ptr()
        arg.out_scores, arg.out_tokens, arg.out_parents, arg.out_done = (values.data_ptr(), tokens.data_ptr(), parents.data_ptr(),
                                                                         over.data_ptr())
        if done is not None:
            arg.done = done.data_ptr()
        rc = _cabi.lib().l3_beam_select(C.byref(arg))
        if rc:
            _cabi.check(rc)
    return values, tokens, parents, over


def _plan_reorder(states, parents):
    _tensor(parents, "parents", 2)
    _ints(parents, "parents", tuple(parents.shape))
    batch, beams = parents.shape
    _need(1 <= beams <= MOST_BEAMS and batch <= 65535, "parents of shape %s: 1 to %d beams of up to 65535 sequences are supported",
          (batch, beams), MOST_BEAMS)
    rows = _rows(states, "states")
    for x in states:
        _need(x.shape[0] == batch * beams, "a state has %d rows for %d x %d beams", x.shape[0], batch, beams)
    device = _one_device([("parents", parents)] + [("states", x) for x in states])
    return bytes(rows), device.index, batch, beams


def beam_reorder(states, parents):
    """In place, row b * beams + j of every state becomes what row b * beams + parents[b, j] was.

    states   a list of tensors [batch * beams, ...] of any type: recurrent states, page tables, token histories, cache rows; a row
             is a contiguous run, or equal runs at equal distances (`cache[:, :, first:last]`)
    parents  [batch, beams] int32, any of a sequence's beams, several times too; a number outside leaves its row as it is
    """
    states = [states] if isinstance(states, torch.Tensor) else list(states)
    try:
        key = (_form(parents), *map(_form, states))
    except (AttributeError, RuntimeError):
        key = None
    fixed, index, batch, beams = _plan_reorder(states, parents) if key is None else _planned(_reorder_plans, key, _plan_reorder, states,
                                                                                             parents)
    if batch:
        rc = _cabi.lib().l3_beam_reorder(index, _stream(index), _filled(fixed, states), len(states), parents.data_ptr(), batch, beams)
        if rc:
            _cabi.check(rc)
