"""A key / value cache in pages: operators on torch CUDA tensors, and `PagedCache`, the bookkeeping of its pages.

The reference has one array per layer, [batch, positions, kv heads, head size], owned by its attention module
(llama3.py:138-153, 184-187).  Here a cache is a pool of pages of a fixed number of tokens; a sequence is a row of a table that
names its pages in order, so that sequences grow without moving and share what they have in common.

Every operator enqueues its kernels on the current stream of the tensors' device and returns; it can be captured into a graph.
Arguments that do not fit raise ValueError before anything is enqueued.  What is in device memory - lengths, tables - is not
read by the host: a page number outside the pool names a page that holds no tokens.

Pools have the dimensions [pages, kv heads, page size, head size] in any memory order whose last dimension is contiguous; a
pool kept as [pages, page size, kv heads, head size] is passed as `pool.transpose(1, 2)`.
"""
from __future__ import annotations

import ctypes as C
import heapq

import torch

from . import _cabi

_KIND = {torch.float32: _cabi.DTYPE_F32, torch.bfloat16: _cabi.DTYPE_BF16, torch.float16: _cabi.DTYPE_F16}
HEAD_DIMS = (16, 32, 48, 64, 96, 128)


def _need(cond, text, *args):
    if not cond:
        raise ValueError(text % args if args else text)


def _tensor(x, name, dims, dtypes=None):
    _need(isinstance(x, torch.Tensor), "%s must be a tensor", name)
    _need(x.dim() == dims, "%s must have %d dimensions, got %s", name, dims, tuple(x.shape))
    if dtypes is not None:
        _need(x.dtype in dtypes, "%s: type %s is not one of %s", name, x.dtype, ", ".join(str(d) for d in dtypes))
    return x


def _ints(x, name, shape):
    _tensor(x, name, len(shape), (torch.int32,))
    _need(tuple(x.shape) == tuple(shape), "%s must be %s, got %s", name, tuple(shape), tuple(x.shape))
    _need(x.is_contiguous(), "%s must be contiguous", name)
    return x


def _one_device(named):
    device = None
    for name, x in named:
        if x is None:
            continue
        _need(x.is_cuda, "%s must be on a CUDA device", name)
        device = x.device if device is None else device
        _need(x.device == device, "%s is on %s, the others on %s", name, x.device, device)
    return device


def _pool(k_pages, v_pages):
    _tensor(k_pages, "k_pages", 4, tuple(_KIND))
    _tensor(v_pages, "v_pages", 4, (k_pages.dtype,))
    _need(k_pages.shape == v_pages.shape, "k_pages and v_pages differ: %s and %s", tuple(k_pages.shape), tuple(v_pages.shape))
    pages, _, page, dim = k_pages.shape
    _need(pages >= 1 and page >= 1 and page & (page - 1) == 0 and page <= 65536, "page size %d is not a power of two up to 65536", page)
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages)):
        _need(x.stride(3) == 1 or dim == 1, "%s: the last dimension must be contiguous", name)
        _fits16(name, x)


def _fits16(name, x):
    size = x.element_size()
    _need(x.data_ptr() % 16 == 0 and all(s * size % 16 == 0 for n, s in zip(x.shape[:-1], x.stride()) if n > 1),
          "%s: addresses must be multiples of 16 bytes", name)


def _strides(x, *dims):
    """Strides in elements; 0 where a dimension has one entry only (its stride may be anything)."""
    return [x.stride(d) if x.shape[d] > 1 else 0 for d in dims]


def _stream(device_index):
    return torch._C._cuda_getCurrentRawStream(device_index)


# A call's checks and the parts of its C struct that hang on shapes, strides, types and the device alone are made once per such
# form: they take several times as long as the kernels of a small call.  Addresses and values are never kept.
_MOST_PLANS = 4096


def _form(x):
    return None if x is None else (x.shape, x.stride(), x.dtype, x.get_device())


def _planned(plans, key, make, *args):
    plan = plans.get(key)
    if plan is None:
        if len(plans) >= _MOST_PLANS:
            plans.clear()
        plan = make(*args)
        plans[key] = plan
    return plan


_attention_plans: dict = {}


def _plan_attention(q, k_pages, v_pages, page_table, lengths, k_new, v_new, scale, out):
    _tensor(q, "q", 3, tuple(_KIND))
    _pool(k_pages, v_pages)
    batch, heads, dim = q.shape
    pages, kv_heads, page, _ = k_pages.shape
    _need(q.dtype in (k_pages.dtype, torch.float32), "q must have the cache's type or fp32, got %s over %s", q.dtype, k_pages.dtype)
    _need(k_pages.shape[3] == dim and dim in HEAD_DIMS, "head size %d (cache: %d) is not one of %s", dim, k_pages.shape[3], HEAD_DIMS)
    _need(kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0, "%d heads over %d kv heads", heads, kv_heads)
    _need(q.stride(2) == 1, "q: the last dimension must be contiguous")
    _tensor(page_table, "page_table", 2, (torch.int32,))
    _need(page_table.shape[0] == batch, "page_table has %d rows for %d sequences", page_table.shape[0], batch)
    _need(page_table.shape[1] <= 1 or page_table.stride(1) == 1, "page_table: a row must be contiguous")
    _ints(lengths, "lengths", (batch,))
    _need((k_new is None) == (v_new is None), "k_new and v_new go together")
    new = [0, 0, 0, 0]
    if k_new is not None:
        for name, x in (("k_new", k_new), ("v_new", v_new)):
            _tensor(x, name, 3, (k_pages.dtype,))
            _need(tuple(x.shape) == (batch, kv_heads, dim), "%s must be %s, got %s", name, (batch, kv_heads, dim), tuple(x.shape))
            _need(x.stride(2) == 1, "%s: the last dimension must be contiguous", name)
            _fits16(name, x)
        new = [*_strides(k_new, 0, 1), *_strides(v_new, 0, 1)]
    if out is not None:
        _tensor(out, "out", 3, (q.dtype,))
        _need(out.shape == q.shape and out.is_contiguous(), "out must be contiguous, of q's shape")
    device = _one_device((("q", q), ("k_pages", k_pages), ("v_pages", v_pages), ("page_table", page_table), ("lengths", lengths),
                          ("k_new", k_new), ("v_new", v_new), ("out", out)))
    n = C.c_int64()
    if batch:
        _cabi.check(_cabi.lib().l3_paged_attention_workspace(device.index, heads, kv_heads, dim, C.byref(n)))
    room = -(-n.value // q.element_size())
    arg = _cabi.L3PagedAttention(
        device.index, batch, heads, kv_heads, dim, pages, page, page_table.shape[1], _KIND[q.dtype], _KIND[k_pages.dtype],
        _KIND[q.dtype], dim ** -0.5 if scale is None else float(scale), None, None, *_strides(q, 0, 1),
        _cabi.L3PagePool(None, *_strides(k_pages, 0, 1, 2)), _cabi.L3PagePool(None, *_strides(v_pages, 0, 1, 2)), None,
        *_strides(page_table, 0), None, None, None, *new, None, None, None, room * q.element_size())
    return bytes(arg), device.index, room, q.is_contiguous(), batch


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
    args = (q, k_pages, v_pages, page_table, lengths, k_new, v_new, scale, out)
    try:
        key = (_form(q), _form(k_pages), _form(v_pages), _form(page_table), _form(lengths), _form(k_new), _form(v_new), scale, _form(out))
    except (AttributeError, RuntimeError):
        key = None                                     # not tensors, or not strided ones: refused below
    fixed, index, room, plain, batch = _plan_attention(*args) if key is None else _planned(_attention_plans, key, _plan_attention, *args)
    if out is None:
        out = torch.empty_like(q) if plain else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = q.new_empty(q.shape[:2], dtype=torch.float32) if return_lse else None
    if batch:
        ws = q.new_empty(room)                         # of this call: a captured graph has one of its own
        arg = _cabi.L3PagedAttention.from_buffer_copy(fixed)
        arg.stream, arg.q, arg.table, arg.lengths = _stream(index), q.data_ptr(), page_table.data_ptr(), lengths.data_ptr()
        arg.k.data, arg.v.data, arg.out, arg.workspace = k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), ws.data_ptr()
        if k_new is not None:
            arg.k_new, arg.v_new = k_new.data_ptr(), v_new.data_ptr()
        if return_lse:
            arg.lse = lse.data_ptr()
        rc = _cabi.lib().l3_paged_attention(C.byref(arg))
        if rc:
            _cabi.check(rc)
    return (out, lse) if return_lse else out


_write_plans: dict = {}


def _plan_write(k, v, k_pages, v_pages, page_table, start, count):
    _pool(k_pages, v_pages)
    pages, kv_heads, page, dim = k_pages.shape
    for name, x in (("k", k), ("v", v)):
        _tensor(x, name, 4, (k_pages.dtype,))
        _need(x.shape == k.shape and tuple(x.shape[2:]) == (kv_heads, dim), "%s must be [batch, tokens, %d, %d], got %s", name, kv_heads,
              dim, tuple(x.shape))
        _need(x.stride(3) == 1 or dim == 1, "%s: the last dimension must be contiguous", name)
        _fits16(name, x)
    _need(dim * k.element_size() % 16 == 0, "head size %d: a head's row must be a multiple of 16 bytes", dim)
    batch, tokens = k.shape[:2]
    _need(batch <= 65535, "at most 65535 sequences a call")
    _tensor(page_table, "page_table", 2, (torch.int32,))
    _need(page_table.shape[0] == batch, "page_table has %d rows for %d sequences", page_table.shape[0], batch)
    _need(page_table.shape[1] <= 1 or page_table.stride(1) == 1, "page_table: a row must be contiguous")
    _ints(start, "start", (batch,))
    if count is not None:
        _ints(count, "count", (batch,))
    device = _one_device((("k", k), ("v", v), ("k_pages", k_pages), ("v_pages", v_pages), ("page_table", page_table), ("start", start),
                          ("count", count)))
    arg = _cabi.L3PagedWrite(
        device.index, batch, tokens, kv_heads, dim, pages, page, page_table.shape[1], _KIND[k.dtype], None, None, None,
        *_strides(k, 0, 1, 2), *_strides(v, 0, 1, 2), _cabi.L3PagePool(None, *_strides(k_pages, 0, 1, 2)),
        _cabi.L3PagePool(None, *_strides(v_pages, 0, 1, 2)), None, *_strides(page_table, 0), None, None)
    return bytes(arg), device.index, batch * tokens


def paged_write(k, v, k_pages, v_pages, page_table, start, count=None):
    """Writes keys and values of a padded batch into their pages.

    k, v   [batch, tokens, kv heads, head size] of the pools' type; token t < count[b] of sequence b becomes its token start[b] + t
    start, count   [batch] int32 (count None: every token is real)
    Tokens that the table has no page for are dropped; what lies behind a sequence's last token stays as it was.
    """
    args = (k, v, k_pages, v_pages, page_table, start, count)
    try:
        key = (_form(k), _form(v), _form(k_pages), _form(v_pages), _form(page_table), _form(start), _form(count))
    except (AttributeError, RuntimeError):
        key = None
    fixed, index, some = _plan_write(*args) if key is None else _planned(_write_plans, key, _plan_write, *args)
    if some:
        arg = _cabi.L3PagedWrite.from_buffer_copy(fixed)
        arg.stream, arg.k, arg.v, arg.table, arg.start = _stream(index), k.data_ptr(), v.data_ptr(), page_table.data_ptr(), start.data_ptr()
        arg.k_pool.data, arg.v_pool.data = k_pages.data_ptr(), v_pages.data_ptr()
        if count is not None:
            arg.count = count.data_ptr()
        rc = _cabi.lib().l3_paged_write(C.byref(arg))
        if rc:
            _cabi.check(rc)


def _rows(tensors, what):
    """L3Rows of tensors whose first dimension counts rows; a row is a contiguous run, or equal runs at equal distances."""
    _need(len(tensors) >= 1, "no %s", what)
    out = (_cabi.L3Rows * len(tensors))()
    for i, x in enumerate(tensors):
        _need(isinstance(x, torch.Tensor) and x.dim() >= 1, "%s must be tensors with rows", what)
        size = x.element_size()
        dims = [(n, s) for n, s in zip(x.shape[1:], x.stride()[1:]) if n != 1]
        if any(n == 0 for n, _ in dims):
            dims = [(0, 1)]
        run, outer, outer_stride = 1, 1, 0
        while dims and dims[-1][1] == run:
            run *= dims.pop()[0]
        if dims:                                  # the next dimensions out, as far as they are one
            outer, outer_stride = dims.pop()
            while dims and dims[-1][1] == outer * outer_stride:
                outer *= dims.pop()[0]
        _need(not dims, "%s %d: a row of shape %s and strides %s is not a run, or equal runs at equal distances", what, i,
              tuple(x.shape[1:]), tuple(x.stride()[1:]))
        row = x.stride(0)
        span = (outer - 1) * outer_stride + run if run and outer else 0
        _need(outer <= 1 or outer_stride >= run, "%s %d overlaps itself", what, i)
        _need(x.shape[0] <= 1 or row >= span or _interleaved(x, row, run, outer, outer_stride), "%s %d: rows overlap", what, i)
        out[i] = _cabi.L3Rows(None, x.shape[0], row * size, outer, outer_stride * size, run * size)
    return out


def _interleaved(x, row, run, outer, outer_stride):
    """Rows that lie between one another's runs, as in a cache kept [heads, sequences, ...]."""
    return run <= row and row * x.shape[0] <= outer_stride


_copy_plans: dict = {}


def _plan_copy(pools, src, dst):
    rows = _rows(pools, "pools")
    for x in pools:
        _need(x.shape[0] == pools[0].shape[0], "pools have %d and %d pages", pools[0].shape[0], x.shape[0])
    _tensor(src, "src", 1)
    _ints(src, "src", (src.shape[0],))
    _ints(dst, "dst", (src.shape[0],))
    device = _one_device([("src", src), ("dst", dst)] + [("pools", x) for x in pools])
    return bytes(rows), device.index


def _filled(fixed, tensors):
    """The L3Rows of a plan, with the tensors' addresses."""
    rows = (_cabi.L3Rows * len(tensors)).from_buffer_copy(fixed)
    for r, x in zip(rows, tensors):
        r.base = x.data_ptr()
    return rows


def copy_pages(pools, src, dst):
    """Page dst[i] becomes a copy of page src[i] in every pool: pools a list of tensors [pages, ...], src and dst [n] int32.

    Pairs with a number outside the pools are skipped.  No page may be a destination twice, nor both source and destination.
    """
    pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    try:
        key = (_form(src), _form(dst), *map(_form, pools))
    except (AttributeError, RuntimeError):
        key = None
    fixed, index = _plan_copy(pools, src, dst) if key is None else _planned(_copy_plans, key, _plan_copy, pools, src, dst)
    n = src.shape[0]
    if n:
        rc = _cabi.lib().l3_copy_rows(index, _stream(index), _filled(fixed, pools), len(pools), src.data_ptr(), dst.data_ptr(), n)
        if rc:
            _cabi.check(rc)


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
        _need(dtype in _KIND, "type %s is not one of %s", dtype, ", ".join(str(d) for d in _KIND))
        self.device = torch.device(device)
        shape = (pages, kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layers)]

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
