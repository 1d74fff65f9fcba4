"""A packed step over a cache in pages: the new tokens of many requests - whole prompts, portions of prompts, single tokens - as the rows of
one batch, on torch CUDA tensors.

    step = paged_extend(table, lengths, counts, free_pages, page_size=16, tokens=rows)   # pages, positions and slots of the new tokens
    for every layer:
        q, k, v = ...                                                                    # [rows, heads, head size]
        q = paged_rotary_write(q, k, v, step.positions, step.slots, k_pages, v_pages, frequencies)
        out = paged_chunk_attention(q, k_pages, v_pages, table, step.lengths, step.starts)
    scores = token_logprobs(logits, tokens, top=5, entropy=True)

The reference has one batch of equal lengths at one position (llama3.py:285-304) and turns queries and keys by precomputed tables
(llama3.py:31-76).  Request b has the rows starts[b] .. starts[b + 1] - 1, its newest tokens in order; rows behind the last request
belong to none, so that a captured graph serves any mixture of up to its number of rows.

Every operator enqueues its kernels on the current stream of the tensors' device and returns; it can be captured into a graph.  Arguments
that do not fit raise ValueError before anything is enqueued.  What is in device memory is not read by the host.  The operators have no
derivatives: outside torch.no_grad() they refuse tensors that require a gradient, and tensors with a forward-mode gradient.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import paged
from .paged import _need


class PackedStep(NamedTuple):
    """What `paged_extend` returns."""
    lengths: torch.Tensor      # [batch] int32: tokens of every request, the new ones among them
    starts: torch.Tensor       # [batch + 1] int32: its rows
    positions: torch.Tensor    # [tokens] int32: of every row; -1 for one of no request
    slots: torch.Tensor        # [tokens] int64: its place in the pools, page * page size + token of the page; -1: none
    used: torch.Tensor         # [1] int32: pages that were needed


class TokenLogprobs(NamedTuple):
    """What `token_logprobs` returns."""
    logprobs: torch.Tensor                  # [rows] fp32
    entropy: Optional[torch.Tensor]         # [rows] fp32
    top_logprobs: Optional[torch.Tensor]    # [rows, top] fp32
    top_tokens: Optional[torch.Tensor]      # [rows, top] int32


def paged_extend(page_table, lengths, counts, free_pages, *, page_size, tokens):
    """A step's bookkeeping on the device: request b has lengths[b] tokens and gets counts[b] more.

    page_table   [batch, max pages] int32; new pages go behind those of the tokens that a request has, in place
    lengths, counts   [batch] int32; negative numbers count as 0
    free_pages   [n] int32: pages to take from, in this order, request by request
    tokens       rows of the step; requests whose tokens do not fit get fewer, the last ones first
    Returns a PackedStep.  More pages used than free_pages has: those that were not there are -1 in the table, and hold no tokens.
    A partly filled last page goes on being filled: pages that requests share are `PagedCache`'s to copy.
    """
    return PackedStep._make((paged._module or paged._ops()).paged_extend(page_table, lengths, counts, free_pages, page_size, tokens))


def rotary_frequencies(dims, base=10000.0, *, kind=None, factor=1.0, original=8192, low=1.0, high=4.0, device="cuda"):
    """Frequencies of rotary positions, base ** (-2 i / dims) radians a position for pair i, [dims / 2] float64, and the amplitude that
    goes with them (1 but for "yarn").

    kind   how positions beyond the `original` ones of training are reached, `factor` times as many:
           None       not at all
           "linear"   every frequency over factor
           "ntk"      base * factor ** (dims / (dims - 2)): the slowest frequency over factor, the fastest as it is
           "llama3"   frequencies of fewer than `low` turns in `original` positions over factor, of more than `high` as they are, between
                      them faded by their turns
           "yarn"     the same by pair: as they are up to the pair of `high` turns, over factor from the pair of `low` turns on, faded in
                      between; amplitude 0.1 log(factor) + 1  (customary: low 1, high 32)
    """
    _need(isinstance(dims, int) and dims >= 2 and dims % 2 == 0, "dims %s: an even number of entries is turned", dims)
    _need(math.isfinite(base) and base > 0, "base %s", base)
    _need(kind in (None, "linear", "ntk", "llama3", "yarn"), "kind %r is not one of None, 'linear', 'ntk', 'llama3', 'yarn'", kind)
    _need(math.isfinite(factor) and factor >= 1, "factor %s is below 1", factor)
    amplitude = 1.0
    if kind == "ntk":
        _need(dims > 2, "kind 'ntk' needs more than one pair")
        base = base * factor ** (dims / (dims - 2))
    i = torch.arange(dims // 2, dtype=torch.float64)
    f = base ** (-2 * i / dims)
    if kind == "linear":
        f = f / factor
    elif kind in ("llama3", "yarn"):
        _need(original >= 1 and 0 < low < high and math.isfinite(high), "original %s, low %s, high %s", original, low, high)
        if kind == "llama3":
            keep = (original * f / (2 * math.pi) - low) / (high - low)
        else:
            _need(base > 1, "kind 'yarn' needs a base above 1")

            def pair(turns):  # the (fractional) pair that makes so many turns in `original` positions
                return dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

            first, last = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), dims - 1)
            keep = 1 - (i - first) / max(last - first, 0.001)
            amplitude = 0.1 * math.log(factor) + 1.0
        keep = keep.clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f.to(device), amplitude


def rotary(x, positions, frequencies, *, layout="pairs", amplitude=1.0, inverse=False, out=None):
    """Turns the first 2 * len(frequencies) entries of every head to its row's position.

    x            [tokens, heads, head size] or [batch, tokens, heads, head size], fp32, bfloat16 or float16, any strides with a
                 contiguous last dimension
    positions    [tokens] or [batch, tokens] int32; a row at a negative one stays as it is
    frequencies  [dims / 2] float64: radians a position (`rotary_frequencies`); angles are taken in 64 bits
    layout       "pairs": entries 2 i and 2 i + 1 belong together (the reference's), "halves": i and i + dims / 2
    amplitude    of what is turned; inverse: by the negative angle
    out          where the result goes; x itself, or memory of its own
    """
    return (paged._module or paged._ops()).rotary(x, positions, frequencies, layout, amplitude, bool(inverse), out)


def paged_rotary_write(q, k, v, positions, slots, k_pages, v_pages, frequencies, *, layout="pairs", amplitude=1.0, out=None):
    """`rotary` of queries and keys, and the keys and values into their slots of the pools, in one launch.

    q            [tokens, heads, head size], k, v [tokens, kv heads, head size], of the pools' type
    slots        [tokens] int64, page * page size + token of the page, no two alike; one outside the pools: the row is written nowhere
    k_pages, v_pages   pools as `paged_attention` takes them
    Returns the turned queries (written into `out` where given: q itself, or memory of its own; never the pools').
    """
    return (paged._module or paged._ops()).paged_rotary_write(q, k, v, positions, slots, k_pages, v_pages, frequencies, layout, amplitude, out)


def paged_chunk_attention(q, k_pages, v_pages, page_table, lengths, starts, *, scale=None, return_lse=False, out=None):
    """Attention of a packed step's rows over the pages of their requests: a row sees its request's tokens up to its own.

    q            [tokens, heads, head size] of the pools' type; query head h reads kv head h // (heads / kv heads)
    k_pages, v_pages   the pools, fp32, bfloat16 or float16, the new tokens written already
    page_table   [batch, max pages] int32; token j of a request is in page `page_table[b, j // page size]`
    lengths      [batch] int32: tokens of a request, the new ones among them
    starts       [batch + 1] int32: request b has the rows starts[b] .. starts[b + 1] - 1, its newest tokens; requests may have none
    scale        of q . k; 1 / sqrt(head size) by default
    Returns [tokens, heads, head size] of q's type (written into `out` where given: memory of its own), and with `return_lse` also the log of the softmax's
    denominator, [tokens, heads] fp32.  A row that sees no token has result 0 and lse -inf.  Rows of no request are left as they are in
    `out`, and 0 in a result that is made here.
    """
    return (paged._module or paged._ops()).paged_chunk_attention(q, k_pages, v_pages, page_table, lengths, starts, scale, bool(return_lse), out)


def token_logprobs(logits, tokens, *, top=0, entropy=False):
    """Log probabilities of given tokens under rows of logits.

    logits  [rows, vocab] fp32, bfloat16 or float16, last dimension contiguous
    tokens  [rows] int32; a negative one is none, its log probability 0, and one beyond the vocabulary has NaN
    top     how many of the most likely tokens come back beside them, up to 64: largest logit first, equal ones by token
    entropy the distribution's, too (in nats)
    Returns a TokenLogprobs.  A token of logit -inf has probability 0; a place of `top` that no other token is left for has the token -1 at
    -inf; a row of such tokens alone has entropy 0; a row with +inf or NaN has NaN.
    """
    return TokenLogprobs._make((paged._module or paged._ops()).token_logprobs(logits, tokens, top, bool(entropy)))
