"""GPU suite: bookkeeping and rotary positions of a packed step, and a run of its operators as a decoder uses them."""
import math
import random

import pytest
import torch

from llama3_np_b200 import (PagedCache, paged_chunk_attention, paged_extend, paged_rotary_write, rotary, rotary_frequencies, token_logprobs)

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


# ------------------------------------------------------------------------------------------------------------ bookkeeping
def extended(table, lengths, counts, free, page, tokens):
    """By the definition, one request after the other."""
    table, wide = [list(r) for r in table], len(table[0]) if table else 0
    at = rows = 0
    new, starts, positions, slots = [], [0], [-1] * tokens, [-1] * tokens
    for b, (n, c) in enumerate(zip(lengths, counts)):
        n, c = max(n, 0), min(max(c, 0), tokens - rows)
        for j in range(-(-n // page), -(-(n + c) // page)):
            if j < wide:
                table[b][j] = free[at] if at < len(free) else -1
            at += 1
        for i in range(c):
            p = n + i
            positions[rows + i] = p
            if p // page < wide and table[b][p // page] >= 0:
                slots[rows + i] = table[b][p // page] * page + p % page
        rows += c
        new.append(n + c)
        starts.append(rows)
    return table, new, starts, positions, slots, at


@pytest.mark.parametrize("page", [1, 4, 16, 64])
@pytest.mark.parametrize("batch,most,longest", [(1, 1, 0), (1, 3000, 70), (5, 40, 100), (33, 1, 900), (400, 30, 200), (511, 3, 50), (513, 9, 60), (3000, 4, 90)])
@pytest.mark.parametrize("trouble", ["", "cut", "pages", "narrow"])
def test_extend(page, batch, most, longest, trouble):
    rng = random.Random(page * batch)
    lengths = [rng.randint(0, longest) if rng.random() < 0.8 else 0 for _ in range(batch)]
    counts = [rng.choice([0, 1, rng.randint(0, most), most]) for _ in range(batch)]
    if batch > 3:
        lengths[1], counts[2] = -4, -3
    need = [-(-(max(n, 0) + max(c, 0)) // page) - -(-max(n, 0) // page) for n, c in zip(lengths, counts)]
    wide = max(-(-(max(n, 0) + max(c, 0)) // page) for n, c in zip(lengths, counts)) + 1
    ids = list(range(sum(-(-max(n, 0) // page) for n in lengths) + sum(need) + 3))
    rng.shuffle(ids)
    table, at = [], 0
    if trouble == "narrow":
        wide = max(wide // 2, 1)
    for n in lengths:
        had = -(-max(n, 0) // page)
        table.append((ids[at:at + had] + [-9] * wide)[:wide])
        at += had
    free = ids[at:]
    if trouble == "pages":
        free = free[:sum(need) // 2]
    rows = sum(max(c, 0) for c in counts)
    tokens = rows * 2 // 3 if trouble == "cut" else rows + rng.choice([0, 5, 700])
    dev = ints(table)
    args = (dev, ints(lengths), ints(counts), ints(free))
    step = paged_extend(*args, page_size=page, tokens=tokens)
    want = extended(table, lengths, counts, free, page, tokens)
    for got, w in zip((dev, *step), want):
        assert torch.equal(got.cpu().long(), torch.tensor(w if isinstance(w, list) else [w]).reshape(got.shape)), (got, w)
    assert step.slots.dtype == torch.int64 and step.positions.dtype == torch.int32
    again = paged_extend(*args, page_size=page, tokens=tokens)   # nothing that it reads has changed
    assert all(torch.equal(a, b) for a, b in zip(step, again))


def test_extend_of_nothing_and_at_the_end_of_the_numbers():
    none = ints([])
    step = paged_extend(ints([]).reshape(0, 3), none, none, none, page_size=8, tokens=4)
    assert step.starts.tolist() == [0] and step.positions.tolist() == [-1] * 4 and step.slots.tolist() == [-1] * 4 and step.used.tolist() == [0]
    step = paged_extend(ints([[5]]), ints([3]), ints([0]), none, page_size=8, tokens=0)
    assert step.lengths.tolist() == [3] and step.starts.tolist() == [0, 0]
    top = 2 ** 31 - 1
    step = paged_extend(ints([[5], [6]]), ints([top, top - 2]), ints([top, top]), ints([]), page_size=8, tokens=5)
    assert step.lengths.tolist() == [top, top] and step.starts.tolist() == [0, 0, 2] and step.positions.tolist() == [top - 2, top - 1, -1, -1, -1]
    step = paged_extend(ints([[2 ** 31 - 1]]), ints([1]), ints([1]), ints([]), page_size=65536, tokens=1)
    assert step.slots.tolist() == [(2 ** 31 - 1) * 65536 + 1]


def test_extend_is_captured_and_goes_on():
    """Three replays of one graph that feeds its lengths and free pages back."""
    table, lengths, counts, free = ints([[-1] * 6] * 3), ints([0, 0, 0]), ints([5, 1, 0]), ints(list(range(20)))
    paged_extend(table.clone(), lengths, counts, free, page_size=4, tokens=8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step = paged_extend(table, lengths, counts, free, page_size=4, tokens=8)
        lengths.copy_(step.lengths)
        at = (torch.arange(20, device="cuda") + step.used).clamp(max=19)
        free.copy_(free[at])
    for _ in range(3):
        g.replay()
    assert lengths.tolist() == [15, 3, 0]
    assert table.tolist() == [[0, 1, 3, 4, -1, -1], [2, -1, -1, -1, -1, -1], [-1] * 6]


# -------------------------------------------------------------------------------------------------------- rotary positions
def turned(x, positions, f, layout, amplitude=1.0, inverse=False):
    """In 64 bits, and a bound of the error ahead of the last rounding: cosine and sine, two products and their sum in fp32."""
    y, d = x.double(), 2 * len(f)
    angle = positions.double()[..., None] * f * (-1 if inverse else 1)
    keep = (positions < 0)[..., None]
    c = torch.where(keep, torch.ones_like(angle), angle.cos() * amplitude)[..., None, :]
    s = torch.where(keep, torch.zeros_like(angle), angle.sin() * amplitude)[..., None, :]
    out, tol = y.clone(), torch.zeros_like(y)
    first = torch.arange(0, d, 2, device="cuda") if layout == "pairs" else torch.arange(d // 2, device="cuda")
    second = first + (1 if layout == "pairs" else d // 2)
    a, b = y[..., first], y[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    tol[..., first] = tol[..., second] = (a.abs() + b.abs()) * max(abs(amplitude), 1.0) * 2.0 ** -21
    return out, tol


def near(got, want):
    want, tol = want
    bound = tol + want.abs() * torch.finfo(got.dtype).eps / 2 + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound.clamp(min=1e-30)).max()):.3f} of the bound"


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("dim,dims", [(64, 64), (128, 128), (128, 32), (48, 48), (96, 24), (80, 20), (20, 6), (7, 2), (130, 130), (256, 64), (9, 0)])
def test_rotary(kind, layout, dim, dims):
    g = torch.Generator(device="cuda").manual_seed(dim + dims)
    f = rotary_frequencies(dims, 500000.0)[0] if dims else torch.zeros(0, dtype=torch.float64, device="cuda")
    for tokens, heads, far in ((1, 3, 10), (37, 5, 100000), (1300, 2, 2 ** 31 - 1)):
        x = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(TYPES[kind])
        p = torch.randint(0, far, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        p[::5] = -1
        near(rotary(x, p, f, layout=layout), turned(x, p, f, layout))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_rotary_of_strided_rows(kind, layout):
    """Fused projections, heads ahead of tokens, rows that begin at any entry, batches; the result where it was, or elsewhere."""
    g = torch.Generator(device="cuda").manual_seed(2)
    f = rotary_frequencies(32)[0]
    for at in (0, 1, 2, 4, 6):
        whole = torch.randn(3, 50, 10 * 64 + 8, generator=g, device="cuda").to(TYPES[kind])
        x = whole[..., at:at + 640].view(3, 50, 10, 64)
        p = torch.randint(0, 9999, (3, 50), generator=g, device="cuda", dtype=torch.int32)
        want = turned(x, p, f, layout)
        near(rotary(x, p, f, layout=layout), want)
        near(rotary(x.transpose(1, 2).contiguous().transpose(1, 2), p, f, layout=layout), want)
        before = whole.clone()
        assert rotary(x, p, f, layout=layout, out=x) is x
        near(x, want)
        whole[..., at:at + 640] = before[..., at:at + 640]
        assert torch.equal(whole, before), "entries beside the rows have changed"


def test_rotary_amplitude_and_inverse():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(200, 4, 64, generator=g, device="cuda")
    p = torch.randint(0, 100000, (200,), generator=g, device="cuda", dtype=torch.int32)
    f, a = rotary_frequencies(64, kind="yarn", factor=16.0, original=4096, high=32.0)
    near(rotary(x, p, f, amplitude=a), turned(x, p, f, "pairs", a))
    near(rotary(x, p, f, inverse=True), turned(x, p, f, "pairs", 1.0, True))
    back = rotary(rotary(x, p, f), p, f, inverse=True)
    assert bool(((back - x).abs() <= 2.0 ** -20 * (x.abs() + 4)).all())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("page,dim,dims", [(16, 64, 64), (1, 48, 24), (128, 128, 128), (8, 24, 10)])
def test_rotary_write(kind, layout, page, dim, dims):
    g = torch.Generator(device="cuda").manual_seed(dim)
    f = rotary_frequencies(dims)[0]
    for tokens in (1, 30, 1500):
        pages = -(-tokens // page) + 4
        qkv = torch.randn(tokens, 10, dim, generator=g, device="cuda").to(TYPES[kind])
        q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
        pools = [torch.randn(pages, 2, page, dim, generator=g, device="cuda").to(TYPES[kind]), torch.randn(pages, page, 2, dim, generator=g, device="cuda").to(TYPES[kind]).transpose(1, 2)]
        p = torch.randint(0, 70000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].contiguous()
        slots[3::7] = -1
        slots[5::7] = pages * page
        kept = (slots >= 0) & (slots < pages * page)
        before = [x.clone() for x in pools]
        got = paged_rotary_write(q, k, v, p, slots, *pools, f, layout=layout)
        near(got, turned(q, p, f, layout))
        at = slots[kept]
        near(pools[0][at // page, :, at % page], [x[kept] for x in turned(k, p, f, layout)])
        assert torch.equal(pools[1][at // page, :, at % page], v[kept])
        rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
        rest[at] = False
        for a, b in zip(pools, before):
            assert torch.equal(a.transpose(1, 2).reshape(pages * page, 2, dim)[rest], b.transpose(1, 2).reshape(pages * page, 2, dim)[rest])
        again = paged_rotary_write(q, k, v, p, slots, *pools, f, layout=layout, out=q)
        assert again is q and torch.equal(q, got)


# ------------------------------------------------------------------------------------------------------- a run of them all
class Decoder:
    """Two layers of 8 heads over 2 kv heads of 32, a feed-forward without gate, random weights; exact() is the whole of it in 64 bits, a
    request at a time, without pages."""
    H, G, D, W, V, LAYERS = 8, 2, 32, 64, 97, 2

    def __init__(self):
        g = torch.Generator(device="cuda").manual_seed(11)

        def w(*s):
            return torch.randn(*s, generator=g, device="cuda") / math.sqrt(s[0])
        self.embed, self.head = w(self.V, self.W) * 8, w(self.W, self.V)
        self.qkv = [w(self.W, (self.H + 2 * self.G) * self.D) for _ in range(self.LAYERS)]
        self.o = [w(self.H * self.D, self.W) for _ in range(self.LAYERS)]
        self.frequencies = rotary_frequencies(self.D, 1000.0)[0]

    def step(self, ids, pools, table, step):
        x = self.embed[ids]
        for (kp, vp), qkv, o in zip(pools, self.qkv, self.o):
            y = (x @ qkv).view(-1, self.H + 2 * self.G, self.D)
            q, k, v = y.split([self.H, self.G, self.G], 1)
            q = paged_rotary_write(q, k, v, step.positions, step.slots, kp, vp, self.frequencies)
            x = x + paged_chunk_attention(q, kp, vp, table, step.lengths, step.starts).flatten(1) @ o
        return x @ self.head

    def exact(self, ids):
        n = len(ids)
        x = self.embed[ids].double()
        p = torch.arange(n, device="cuda")
        for qkv, o in zip(self.qkv, self.o):
            y = (x @ qkv.double()).view(n, self.H + 2 * self.G, self.D)
            q, k, v = y.split([self.H, self.G, self.G], 1)
            q, k = turned(q, p, self.frequencies, "pairs")[0], turned(k, p, self.frequencies, "pairs")[0]
            k, v = (t.repeat_interleave(self.H // self.G, 1) for t in (k, v))
            s = torch.einsum("thd,khd->htk", q, k) / math.sqrt(self.D)
            s = s.masked_fill(p[None, :] > p[:, None], -math.inf)
            x = x + torch.einsum("htk,khd->thd", torch.softmax(s, -1), v).flatten(1) @ o.double()
        return torch.log_softmax(x @ self.head.double(), -1)


def test_a_run_of_all_of_them():
    """Portions of prompts beside single tokens, over seven captured steps: each token's log probability, and the pages, are what the requests alone have."""
    net, page, rows = Decoder(), 8, 40
    rng = random.Random(4)
    texts = [[rng.randrange(net.V) for _ in range(n)] for n in (90, 3, 17, 64)]
    portions = [[33, 30, 20, 4, 1, 1, 1], [1, 1, 1, 0, 0, 0, 0], [0, 0, 16, 1, 0, 0, 0], [6, 9, 0, 30, 11, 7, 1]]
    pools = [[torch.full((40, net.G, page, net.D), math.nan, device="cuda") for _ in range(2)] for _ in range(net.LAYERS)]
    table, lengths, free = ints([[-1] * 13] * 4), ints([0] * 4), ints(rng.sample(range(40), 40))
    ids, nexts, counts = torch.zeros(rows, dtype=torch.long, device="cuda"), ints([-1] * rows), ints([1, 1, 1, 1])

    def one():
        step = paged_extend(table, lengths, counts, free, page_size=page, tokens=rows)
        logits = net.step(ids, pools, table, step)
        got = token_logprobs(logits, nexts, top=3, entropy=True)
        lengths.copy_(step.lengths)
        free.copy_(free[(torch.arange(40, device="cuda") + step.used).clamp(max=39)])
        return step, got
    with torch.no_grad():
        saved = [t.clone() for t in (table, lengths, free)]
        one()
        for t, s in zip((table, lengths, free), saved):
            t.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step, got = one()
        seen, exact = [0] * 4, [net.exact(torch.tensor(t, device="cuda")) for t in texts]
        for i in range(7):
            n = [p[i] for p in portions]
            ids.zero_(), nexts.fill_(-1)
            at = 0
            for b, c in enumerate(n):
                ids[at:at + c] = torch.tensor(texts[b][seen[b]:seen[b] + c], dtype=torch.long)
                more = (texts[b] + [-1])[seen[b] + 1:seen[b] + 1 + c]
                nexts[at:at + c] = torch.tensor(more, dtype=torch.int32)
                at += c
            counts.copy_(ints(n))
            graph.replay()
            assert int(step.used) <= 40 and step.starts.tolist()[-1] == at
            row = 0
            for b, c in enumerate(n):
                want = exact[b][seen[b]:seen[b] + c]
                for j in range(c):
                    token = int(nexts[row])
                    if token >= 0:
                        assert abs(float(got.logprobs[row]) - float(want[j, token])) < 1e-4
                    else:
                        assert float(got.logprobs[row]) == 0
                    assert abs(float(got.entropy[row]) + float((want[j].exp() * want[j]).sum())) < 1e-4
                    assert torch.allclose(got.top_logprobs[row].double(), want[j].sort(descending=True).values[:3], atol=1e-4, rtol=0)
                    row += 1
                seen[b] += c
        assert seen == [90, 3, 17, 57 + 7]


def test_a_cache_of_pages_has_them():
    """PagedCache.extend and its view beside paged_extend: the same places."""
    cache = PagedCache(layers=1, kv_heads=2, head_dim=32, pages=30, page_size=8, dtype=torch.float32)
    a, b = cache.open(), cache.open()
    cache.extend([a, b], [13, 4])
    for pool in (cache.k[0], cache.v[0]):
        pool.normal_()
    view = cache.extend([a, b], [20, 1])
    q, k, v = (torch.randn(21, n, 32, device="cuda") for n in (4, 2, 2))
    f = rotary_frequencies(32)[0]
    got = cache.attend_packed(0, view, cache.write_packed(0, view, q, k, v, f))
    assert view.starts.tolist() == [0, 20, 21] and view.positions.tolist() == list(range(13, 33)) + [4]
    at = [int(view.table[0, p // 8]) * 8 + p % 8 for p in range(13, 33)] + [int(view.table[1, 0]) * 8 + 4]
    assert view.slots.tolist() == at
    kp, vp = cache.k[0].clone(), cache.v[0].clone()
    want = paged_chunk_attention(paged_rotary_write(q, k, v, view.positions, view.slots, kp, vp, f), kp, vp, view.table, view.lengths, view.starts)
    assert torch.equal(got, want) and torch.equal(kp, cache.k[0])
    assert view.slots is view.slots and cache.view([a]).positions.tolist() == []
