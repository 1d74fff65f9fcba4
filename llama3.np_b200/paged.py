"""A key / value cache in pages: operators on torch CUDA tensors, and `PagedCache`, the bookkeeping of its pages.

The reference has one array per layer, [batch, positions, kv heads, head size], owned by its attention module
(llama3.py:138-153, 184-187).  Here a cache is a pool of pages of a fixed number of tokens; a sequence is a row of a table that
names its pages in order, so that sequences grow without moving and share what they have in common.

Every operator enqueues its kernels on the current stream of the tensors' device and returns; it can be captured into a graph.
Arguments that do not fit raise ValueError before anything is enqueued.  What is in device memory - lengths, tables - is not
read by the host: a page number outside the pool names a page that holds no tokens.

The operators have no derivatives: outside torch.no_grad() they refuse tensors that require a gradient, and tensors with a
forward-mode gradient.

Pools have the dimensions [pages, kv heads, page size, head size] in any memory order whose last dimension is contiguous; a
pool kept as [pages, page size, kv heads, head size] is passed as `pool.transpose(1, 2)`.
"""
from __future__ import annotations

import ctypes as C
import heapq
import importlib.util
import os

import torch

from . import _cabi

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
HEAD_DIMS = (16, 32, 48, 64, 96, 128)
_module = None


def _ops():
    """The calls of csrc/torch_ops.cpp, bound to the library's entries."""
    global _module
    if _module is None:
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_torch_ops.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with `python llama3.np_b200/build.py` (there is no CPU fallback)")
        spec = importlib.util.spec_from_file_location("_torch_ops", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        lib = _cabi.lib()
        module.bind(*(C.cast(getattr(lib, name), C.c_void_p).value for name in (
            "l3_paged_attention_workspace", "l3_paged_attention", "l3_paged_write", "l3_copy_rows", "l3_beam_reorder",
            "l3_beam_select_workspace", "l3_beam_select", "l3_last_error")))
        _module = module
    return _module


def _need(cond, text, *args):
    if not cond:
        raise ValueError(text % args if args else text)


def paged_attention(q, k_pages, v_pages, page_table, lengths, *, k_new=None, v_new=None, scale=None, return_lse=False, out=None):
    """Attention of one token per sequence over the tokens of its pages.

    q            [batch, heads, head size], the cache's type or fp32; query head h reads kv head h // (heads / kv heads)
    k_pages, v_pages   the pools, fp32, bfloat16 or float16
    page_table   [batch, max pages] int32; token j of a sequence is in page `page_table[b, j // page size]`
    lengths      [batch] int32: tokens that the query sees.  0: the result is 0 (lse -inf)
    k_new, v_new [batch, kv heads, head size]: the newest token, number lengths - 1; used here and written to its page, which no
                 other sequence of the call may share
    scale        of q . k; 1 / sqrt(head size) by default
    Returns [batch, heads, head size] of q's type (written into `out` where given), and with `return_lse` also the log of the
    softmax's denominator, [batch, heads] fp32.
    """
    return (_module or _ops()).paged_attention(q, k_pages, v_pages, page_table, lengths, k_new, v_new, scale, bool(return_lse), out)


def paged_write(k, v, k_pages, v_pages, page_table, start, count=None):
    """Writes keys and values of a padded batch into their pages.

    k, v   [batch, tokens, kv heads, head size] of the pools' type; token t < count[b] of sequence b becomes its token start[b] + t
    start, count   [batch] int32 (count None: every token is real)
    Tokens that the table has no page for are dropped; what lies behind a sequence's last token stays as it was.  No two sequences
    of a call may write to the same page's place.
    """
    (_module or _ops()).paged_write(k, v, k_pages, v_pages, page_table, start, count)


def copy_pages(pools, src, dst):
    """Page dst[i] becomes a copy of page src[i] in every pool: pools a list of tensors [pages, ...], src and dst [n] int32.

    Pairs with a number outside the pools are skipped.  No page may be a destination twice, nor both source and destination.
    """
    (_module or _ops()).copy_pages(pools, src, dst)


class PageTable:
    """Which pages hold which tokens: the bookkeeping of a cache in pages, on the host, without the pages themselves.

    A sequence is a list of pages and a length.  Pages are shared (`fork`) and counted; who adds tokens to a shared, partly filled page
    gets a page of its own first.  Calls that need pages copied return the pairs `(source, destination)`, for `copy_pages`; the new
    state holds once they are copied.  A call that finds too few pages raises RuntimeError and changes nothing."""

    def __init__(self, pages: int, page_size: int):
        _need(pages >= 1, "a cache needs at least one page")
        _need(page_size >= 1 and page_size & (page_size - 1) == 0 and page_size <= 65536, "page size %d is not a power of two up to 65536", page_size)
        self.pages, self.page_size = pages, page_size
        self._free = list(range(pages))     # a heap: the lowest first
        self._refs = [0] * pages
        self._rows: dict = {}               # sequence -> its pages, in order
        self._lengths: dict = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def __contains__(self, seq) -> bool:
        return seq in self._rows

    def _known(self, seq):
        _need(seq in self._rows, "no sequence %s", seq)
        return seq

    def length(self, seq) -> int:
        return self._lengths[self._known(seq)]

    def pages_of(self, seq) -> list:
        return list(self._rows[self._known(seq)])

    def open(self) -> int:
        """A new sequence without tokens."""
        seq, self._next = self._next, self._next + 1
        self._rows[seq], self._lengths[seq] = [], 0
        return seq

    def fork(self, seq) -> int:
        """A new sequence with the same tokens; it shares all pages."""
        self._known(seq)
        new = self.open()
        self._rows[new], self._lengths[new] = list(self._rows[seq]), self._lengths[seq]
        for p in self._rows[new]:
            self._refs[p] += 1
        return new

    def free(self, seq) -> None:
        """Forgets a sequence; pages that no other one shares are free again."""
        for p in self._rows.pop(self._known(seq)):
            self._refs[p] -= 1
            if self._refs[p] == 0:
                heapq.heappush(self._free, p)
        del self._lengths[seq]

    def grow(self, seqs, tokens=1) -> list:
        """Room for `tokens` more tokens (one number, or one of each sequence), which count from now on."""
        seqs = list(seqs)
        more = [tokens] * len(seqs) if isinstance(tokens, int) else list(tokens)
        _need(len(more) == len(seqs) and len(set(seqs)) == len(seqs), "one number of tokens for each sequence, and each sequence once")
        for s, n in zip(seqs, more):
            self._known(s)
            _need(n >= 0, "%s tokens", n)
        # what it takes: new pages, and an own copy of a partly filled page for every sharer but the last
        refs, need = {}, 0
        for s, n in zip(seqs, more):
            row, length = self._rows[s], self._lengths[s]
            need += -(-(length + n) // self.page_size) - len(row)
            if n and length % self.page_size:
                p = row[-1]
                refs.setdefault(p, self._refs[p])
                if refs[p] > 1:
                    refs[p] -= 1
                    need += 1
        if need > len(self._free):
            raise RuntimeError("out of pages: %d needed, %d free" % (need, len(self._free)))
        copies = []
        for s, n in zip(seqs, more):
            row, length = self._rows[s], self._lengths[s]
            if n and length % self.page_size and self._refs[row[-1]] > 1:
                p = self._take()
                self._refs[row[-1]] -= 1
                copies.append((row[-1], p))
                row[-1] = p
            while len(row) * self.page_size < length + n:
                row.append(self._take())
            self._lengths[s] = length + n
        return copies

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._refs[p] = 1
        return p

    def compact(self) -> list:
        """Moves the pages in use to the lowest numbers."""
        used = [p for p in range(self.pages) if self._refs[p]]
        holes = [p for p in range(len(used)) if not self._refs[p]]
        moves = dict(zip((p for p in reversed(used) if p >= len(used)), holes))
        for src, dst in moves.items():
            self._refs[dst], self._refs[src] = self._refs[src], 0
        for row in self._rows.values():
            row[:] = [moves.get(p, p) for p in row]
        self._free = list(range(len(used), self.pages))
        return list(moves.items())


class PagedCache(PageTable):
    """Keys and values of a model's layers in pages, with their bookkeeping.

        cache = PagedCache(layers=32, kv_heads=8, head_dim=128, pages=4096)
        seq = cache.open()
        view = cache.extend([seq], 700)                       # room for a prompt
        cache.write(layer, view, k, v)                        # [1, 700, 8, 128], for every layer
        beams = [seq] + [cache.fork(seq) for _ in range(3)]   # the prompt is shared
        view = cache.extend(beams)                            # one more token each; a shared, partly filled page is copied first
        out = cache.attend(layer, view, q, k_new, v_new)      # [4, heads, 128], for every layer
        cache.free(seq)

    Everything runs on the current stream of the cache's device: a page that is freed and taken again is written behind what read
    it before.  A view is good until the next call that changes one of its sequences, or compacts."""

    class View:
        """Sequences of a cache as its operators take them: `table` [n, pages], `lengths` and `start` [n], int32 on the device; the
        tokens from start on are the newest."""

        def __init__(self, seqs, table, lengths, start):
            self.seqs, self.table, self.lengths, self.start = seqs, table, lengths, start

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page_size: int = 16, dtype=torch.bfloat16, device="cuda"):
        super().__init__(pages, page_size)
        _need(layers >= 1 and kv_heads >= 1, "%d layers of %d kv heads", layers, kv_heads)
        _need(head_dim in HEAD_DIMS, "head size %d is not one of %s", head_dim, HEAD_DIMS)
        _need(dtype in _TYPES, "type %s is not one of %s", dtype, ", ".join(str(d) for d in _TYPES))
        self.device = torch.device(device)
        shape = (pages, kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layers)]
        self.device = self.k[0].device  # "cuda" is a device of its own now, whichever is current later

    def _copy(self, pairs) -> None:
        if pairs:
            both = torch.tensor(pairs, dtype=torch.int32, device=self.device).t().contiguous()
            copy_pages(self.k + self.v, both[0], both[1])

    def view(self, seqs, start=None) -> "PagedCache.View":
        rows, lengths = [self.pages_of(s) for s in seqs], [self.length(s) for s in seqs]
        wide = max((len(r) for r in rows), default=0)
        flat = torch.tensor([r + [-1] * (wide - len(r)) for r in rows], dtype=torch.int32).reshape(len(rows), wide)
        ends = torch.tensor([lengths, lengths if start is None else start], dtype=torch.int32).to(self.device)
        return PagedCache.View(list(seqs), flat.to(self.device), ends[0], ends[1])

    def extend(self, seqs, tokens=1) -> "PagedCache.View":
        """`grow`, with the copies that it takes, and the sequences' view: their new tokens are still to be written (`write`, `attend`)."""
        seqs = list(seqs)
        start = [self.length(s) for s in seqs]
        self._copy(self.grow(seqs, tokens))
        return self.view(seqs, start)

    def compact(self) -> list:
        moves = super().compact()
        self._copy(moves)
        return moves

    def write(self, layer: int, view, k, v) -> None:
        """The view's newest tokens, [sequences, tokens, kv heads, head size], padded where sequences have fewer than others."""
        paged_write(k, v, self.k[layer], self.v[layer], view.table, view.start, (view.lengths - view.start))

    def attend(self, layer: int, view, q, k_new=None, v_new=None, **options):
        """`paged_attention` of the view's sequences over a layer; with k_new and v_new, the newest token of each is written, too."""
        return paged_attention(q, self.k[layer], self.v[layer], view.table, view.lengths, k_new=k_new, v_new=v_new, **options)
