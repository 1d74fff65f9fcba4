"""GPU suite: attention over a cache in pages, writing into it and copying its pages, against their formulas in 64 bits."""
import math

import pytest
import torch

from llama3_np_b200 import copy_pages, paged_attention, paged_write

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(seed, dtype, heads, kv_heads, dim, page, lens, max_pages=None, spare=2, garbage=None, layout="heads"):
    """Pools, a table of pages in random order and lengths; places that no length reaches hold `garbage`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    total = sum(need) + spare
    wide = max(need + [1]) if max_pages is None else max_pages
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), wide), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :min(n, wide)] = torch.tensor(order[at:at + n], dtype=torch.int32)[:wide]
        at += n
    shape = (total, kv_heads, page, dim) if layout == "heads" else (total, page, kv_heads, dim)
    k = torch.randn(shape, generator=g, device="cuda").to(dtype)
    v = torch.randn(shape, generator=g, device="cuda").to(dtype)
    if layout != "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    if garbage is not None:
        used = torch.zeros(total, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(min(n, wide * page)):
                used[table[b, j // page], j % page] = True
        k.masked_fill_(~used.cuda()[:, None, :, None], garbage)
        v.masked_fill_(~used.cuda()[:, None, :, None], garbage)
    q = torch.randn(len(lens), heads, dim, generator=g, device="cuda")
    return q, k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def formula(q, k, v, table, lens, scale=None):
    """(out, lse, error bounds of both ahead of the last rounding) in 64 bits, sequence by sequence."""
    B, H, D = q.shape
    G, page = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    tol = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    tol_lse = torch.zeros(B, H, dtype=torch.float64, device="cuda")
    rows = table.cpu()
    # a weight enters with 16 (bf16: two parts of 8 bits and a sign each) or 22 bits; fp32 as it is
    part = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -21, torch.float32: 0.0}[k.dtype]
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * page))
        pos = [j for j in range(n) if 0 <= int(rows[b, j // page]) < k.shape[0]]
        if not pos:
            continue
        ids = torch.tensor([int(rows[b, j // page]) for j in pos], device="cuda")
        off = torch.tensor([j % page for j in pos], device="cuda")
        for g in range(G):
            hs = slice(g * (H // G), (g + 1) * (H // G))
            kk, vv, qq = k[ids, g, off].double(), v[ids, g, off].double(), q[b, hs].double()
            s = qq @ kk.T * scale
            w = torch.softmax(s, -1)
            out[b, hs], lse[b, hs] = w @ vv, torch.logsumexp(s, -1)
            # scores: D products summed in fp32 (tensor cores may cut instead of round: a step of 2^-22 each), an fp32 query over a 16-bit
            # cache in two 16-bit parts; exponentials 2^-21 and what the argument's last bit makes of it; sums of n / 16 tiles and the join
            es = (qq.abs() @ kk.abs().T).amax(-1) * abs(scale) * ((D + 2) * 2.0 ** -22 + (part if q.dtype != k.dtype else 0))
            delta = 2 * (es + s.abs().amax(-1) * 2.0 ** -22 + 2.0 ** -20 + part) + (len(pos) / 16 + 64) * 2.0 ** -22
            tol[b, hs], tol_lse[b, hs] = delta[:, None] * (w @ vv.abs()), delta
    return out, lse, tol, tol_lse


def check(q, k, v, table, lens, scale=None, **kw):
    got, lse = paged_attention(q, k, v, table, lens, scale=scale, return_lse=True, **kw)
    want, want_lse, tol, tol_lse = formula(q, k, v, table, lens, scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    err = (got.double() - want).abs()
    bound = tol + want.abs() * torch.finfo(q.dtype).eps / 2 + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    assert bool((err <= bound).all()), f"worst {float((err / bound.clamp(min=1e-30)).max()):.3f} of the bound"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    lse_tol = tol_lse + want_lse.abs() * 2.0 ** -23
    assert bool(((lse.double() - want_lse).abs()[~empty] <= lse_tol[~empty]).all())
    return got


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(6, 6), (8, 1), (6, 2), (28, 2), (20, 4)])
@pytest.mark.parametrize("wide", [None, 4000])   # pages a row: a table of few and one of many, over which all warps share all items
def test_shapes(kind, dim, heads, kv_heads, wide):
    lens = [37, 1, 0, 16, 150, 17, 300]
    q, k, v, table, n = make(dim + heads, TYPES[kind], heads, kv_heads, dim, 16, lens, garbage=math.nan, max_pages=wide)
    check(q.to(TYPES[kind]), k, v, table, n)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 64, 256])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("wide", [None, 60000])
def test_pages_and_layouts(kind, page, layout, wide):
    lens = [page, page + 1, max(page - 1, 0), 100, 15, 16, 17, 257]
    q, k, v, table, n = make(page, TYPES[kind], 8, 2, 64, page, lens, garbage=math.inf, layout=layout, max_pages=wide and wide // page)
    check(q.to(TYPES[kind]), k, v, table, n)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [48, 128])
@pytest.mark.parametrize("wide", [None, 4000])
def test_fp32_query_over_16_bit_cache(kind, dim, wide):
    q, k, v, table, n = make(5, TYPES[kind], 12, 3, dim, 16, [5, 700, 64, 33], max_pages=wide)
    check(q, k, v, table, n)
    check(q, k, v, table, n, scale=-0.3)
    assert torch.equal(paged_attention(q, k, v, table, n, scale=0.0), paged_attention(q * 2, k, v, table, n, scale=0.0))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("batch,longest", [(1, 1), (1, 500), (1, 9001), (2, 2500), (5, 900), (20, 300), (70, 60), (300, 40), (1500, 20)])
def test_split_and_joined(kind, batch, longest):
    """From one sequence over all SMs to more items than warps."""
    lens = [1 + (longest - 1) * ((b * 37) % 101) // 100 if b else longest for b in range(batch)]
    q, k, v, table, n = make(batch, TYPES[kind], 4, 2, 64, 16, lens)
    q = q.to(TYPES[kind])
    got = check(q, k, v, table, n)
    assert torch.equal(got, paged_attention(q, k, v, table, n)), "results change from run to run"


@pytest.mark.parametrize("tokens", [64, 20000])
def test_lengths_beyond_the_table_and_below_zero(tokens):
    q, k, v, table, n = make(3, torch.bfloat16, 4, 2, 64, 16, [tokens] * 4)
    q = q.bfloat16()
    n.copy_(torch.tensor([2 * tokens, -5, tokens + 1, tokens], dtype=torch.int32))
    got = check(q, k, v, table, n)
    assert not got[1].any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("wide", [None, 8000])
def test_pages_that_are_not_there(kind, wide):
    q, k, v, table, n = make(4, TYPES[kind], 8, 2, 64, 8, [80, 33, 16, 8], max_pages=wide)
    table[0, 0], table[0, 4], table[1, 1], table[3, 0] = -1, k.shape[0], 1 << 30, -(1 << 31)
    table[2, :2] = -7
    got = check(q.to(TYPES[kind]), k, v, table, n)
    assert not got[2:].any()


def test_no_pages_at_all():
    q, k, v, table, n = make(4, torch.float32, 4, 2, 32, 8, [8, 8])
    got, lse = paged_attention(q, k, v, table[:, :0], n, return_lse=True)
    assert not got.any() and bool((lse == -math.inf).all())
    assert paged_attention(q[:0], k, v, table[:0], n[:0]).shape == (0, 4, 32)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (6, 6, 48, 4), (24, 2, 64, 32)])
@pytest.mark.parametrize("wide", [None, 60000])
def test_new_token(kind, heads, kv_heads, dim, page, wide):
    """The new token's row is used and written; nothing else changes."""
    lens = [1, 16, 17, 0, 100, 33, 260]
    q, k, v, table, n = make(dim, TYPES[kind], heads, kv_heads, dim, page, lens, garbage=math.nan, max_pages=wide and wide // page)
    q = q.to(TYPES[kind])
    new = torch.randn(2, len(lens), kv_heads, dim + 16, device="cuda").to(TYPES[kind])[..., :dim]
    want_k, want_v = k.clone(), v.clone()
    for b, m in enumerate(lens):
        if m:
            p = int(table[b, (m - 1) // page])
            want_k[p, :, (m - 1) % page], want_v[p, :, (m - 1) % page] = new[0, b], new[1, b]
            k[p, :, (m - 1) % page], v[p, :, (m - 1) % page] = math.nan, math.nan
    got = paged_attention(q, k, v, table, n, k_new=new[0], v_new=new[1])
    for x, y in ((k, want_k), (v, want_v)):
        assert torch.equal(x.nan_to_num(7.5), y.nan_to_num(7.5))
    assert torch.equal(got, check(q, want_k, want_v, table, n))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim,page", [(48, 16), (128, 4)])
@pytest.mark.parametrize("batch,longest", [(100, 60), (300, 60), (700, 60), (1900, 30), (300, 250), (16, 300), (60, 250)])
def test_ways_to_share_items(kind, dim, page, batch, longest):
    """Items to a cluster, to a block, to two warps, to one and more than there are warps; new tokens, and sequences without any."""
    lens = [(longest * ((b * 37) % 101) + 99) // 100 if b else longest for b in range(batch)]
    q, k, v, table, n = make(batch + dim, TYPES[kind], 6, 2, dim, page, lens, garbage=math.nan)
    q = q.to(TYPES[kind])
    new = torch.randn(2, batch, 2, dim, device="cuda").to(TYPES[kind])
    b = torch.arange(batch, device="cuda")[n > 0]
    last = n.long()[b] - 1
    p, at = table.long()[b, last // page], last % page
    want_k, want_v = k.clone(), v.clone()
    want_k[p, :, at], want_v[p, :, at] = new[0, b], new[1, b]
    k[p, :, at], v[p, :, at] = math.nan, math.nan
    got = paged_attention(q, k, v, table, n, k_new=new[0], v_new=new[1])
    for x, y in ((k, want_k), (v, want_v)):
        assert torch.equal(x.nan_to_num(7.5), y.nan_to_num(7.5))
    assert torch.equal(got, check(q, want_k, want_v, table, n))


def test_new_token_without_a_page_is_dropped():
    q, k, v, table, n = make(9, torch.bfloat16, 4, 2, 64, 16, [20, 20])
    table[0, 1] = -1
    before = k.clone(), v.clone()
    n[1] = 33                                             # behind the table: cut to it, and written nowhere
    new = torch.randn(2, 2, 2, 64, device="cuda").bfloat16()
    got = paged_attention(q.bfloat16(), k, v, table, n, k_new=new[0], v_new=new[1])
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    want, _, _, _ = formula(q.bfloat16(), k, v, table, n)
    assert float((got.double() - want).abs().max()) < 2.0 ** -6


def test_values_at_the_ends_of_the_range():
    """Large scores: the largest key takes all; equal scores share; a masked place may hold anything."""
    q, k, v, table, n = make(11, torch.bfloat16, 4, 2, 64, 16, [50, 50], garbage=math.nan)
    check((q * 300).bfloat16(), k, v, table, n)
    check((q * 0).bfloat16(), k, v, table, n)
    check(q.bfloat16(), k, (v.float() * 1e30).bfloat16(), table, n)


def test_strided_query_table_and_out():
    q, k, v, table, n = make(12, torch.float16, 8, 4, 96, 16, [30, 90, 1])
    wide = torch.zeros(3, table.shape[1] + 5, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    qw = torch.zeros(3, 8, 200, device="cuda", dtype=torch.float16)
    qw[..., 100:196] = q
    out = torch.empty(3, 8, 96, device="cuda", dtype=torch.float16)
    got = paged_attention(qw[..., 100:196], k, v, wide[:, 2:2 + table.shape[1]], n, out=out)
    assert got is out and torch.equal(out, paged_attention(q.half(), k, v, table, n))


def test_offsets_beyond_32_bits():
    """A pool of 2.3 billion values; the sequence's pages lie at both ends."""
    total, page, G, D = 70000, 64, 4, 128
    k = torch.zeros(total, G, page, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(total, G, page, D, dtype=torch.bfloat16, device="cuda")
    assert k.numel() > 1 << 31
    ids = [0, total - 1, total // 2, total - 2]
    for i in ids:
        k[i], v[i] = torch.randn(G, page, D, device="cuda").bfloat16(), torch.randn(G, page, D, device="cuda").bfloat16()
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    n = torch.tensor([4 * page - 3], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 8, D, device="cuda").bfloat16()
    check(q, k, v, table, n)
    copy_pages([k, v], torch.tensor([total - 1], dtype=torch.int32, device="cuda"), torch.tensor([total - 3], dtype=torch.int32, device="cuda"))
    assert torch.equal(k[total - 3], k[total - 1]) and torch.equal(v[total - 3], v[total - 1])
    row = torch.randn(2, 1, 2, G, D, device="cuda").bfloat16()
    paged_write(row[0], row[1], k, v, torch.tensor([[5, total - 4]], dtype=torch.int32, device="cuda"), torch.tensor([63], dtype=torch.int32, device="cuda"))
    assert torch.equal(k[total - 4, :, 0], row[0, 0, 1]) and torch.equal(v[5, :, 63], row[1, 0, 0])


@pytest.mark.parametrize("wide", [None, 4000])
def test_streams_and_graphs(wide):
    """On a side stream, and captured: two graphs replayed at the same time have workspaces of their own."""
    a = make(21, torch.bfloat16, 8, 2, 128, 16, [900, 300], max_pages=wide)
    b = make(22, torch.bfloat16, 8, 2, 128, 16, [500, 1200], max_pages=wide)
    qs = [x[0].bfloat16() for x in (a, b)]
    want = [paged_attention(q, *x[1:]) for q, x in zip(qs, (a, b))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(paged_attention(qs[0], *a[1:]), want[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for q, x in zip(qs, (a, b)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(paged_attention(q, *x[1:]))
        graphs.append(g)
    for _ in range(20):
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    a[4].fill_(100)                       # lengths are read when the graph runs
    graphs[0].replay()
    assert torch.equal(outs[0], paged_attention(qs[0], *a[1:]))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("tokens,kv_heads,dim,page", [(1, 8, 128, 16), (33, 2, 64, 8), (100, 1, 16, 1), (7, 6, 48, 4), (300, 3, 96, 64)])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_write(kind, tokens, kv_heads, dim, page, layout):
    B, dtype = 5, TYPES[kind]
    start = [0, 3, page, 2 * page - 1, 40]
    count = [tokens, 0, max(1, tokens // 2), tokens, min(tokens, 5)]
    _, kp, vp, table, _ = make(tokens, dtype, kv_heads, kv_heads, dim, page, [s + tokens for s in start], layout=layout)
    table[3, -1] = -1 if tokens > 1 else table[3, -1]
    k = torch.randn(B, tokens, kv_heads, dim, device="cuda").to(dtype)
    v = torch.randn(B, kv_heads, tokens, dim, device="cuda").to(dtype).transpose(1, 2)
    want = kp.clone(), vp.clone()
    rows = table.cpu()
    for b in range(B):
        for t in range(count[b]):
            p = int(rows[b, (start[b] + t) // page])
            if p >= 0:
                want[0][p, :, (start[b] + t) % page], want[1][p, :, (start[b] + t) % page] = k[b, t], v[b, t]
    paged_write(k, v, kp, vp, table, torch.tensor(start, dtype=torch.int32, device="cuda"), torch.tensor(count, dtype=torch.int32, device="cuda"))
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def test_write_drops_what_has_no_place():
    _, kp, vp, table, _ = make(1, torch.float32, 2, 2, 16, 4, [8, 8, 8])
    before = kp.clone(), vp.clone()
    k = torch.randn(3, 6, 2, 16, device="cuda")
    start = torch.tensor([-6, 8, 1 << 30], dtype=torch.int32, device="cuda")
    paged_write(k, k, kp, vp, table, start)
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])
    paged_write(k, k, kp, vp, table, torch.full((3,), 5, dtype=torch.int32, device="cuda"), torch.full((3,), 1000, dtype=torch.int32, device="cuda"))
    p = int(table[1, 1])
    assert torch.equal(kp[p, :, 1:], k[1, :3].transpose(0, 1)) and torch.equal(kp[p, :, 0], before[0][p, :, 0])


@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (40, 8, 16, 128)), (torch.float32, (40, 3, 5)), (torch.uint8, (40, 7)),
                                         (torch.int16, (40, 33)), (torch.float32, (40,)), (torch.bfloat16, (40, 2, 4, 1000))])
@pytest.mark.parametrize("tensors", [1, 3, 70])
def test_copy(dtype, shape, tensors):
    pools = [torch.randint(0, 100, shape, device="cuda").to(dtype) for _ in range(tensors)]
    ids = torch.randperm(40, generator=torch.Generator().manual_seed(3))
    src, dst = ids[:15].int().cuda(), ids[15:30].int().cuda()
    src[3], dst[5], src[7], dst[9] = -1, -1, 40, 1 << 30
    want = [p.clone() for p in pools]
    for w in want:
        for s, d in zip(src.tolist(), dst.tolist()):
            if 0 <= s < 40 and 0 <= d < 40:
                w[d] = w[s]
    copy_pages(pools, src, dst)
    assert all(torch.equal(p, w) for p, w in zip(pools, want))
    copy_pages(pools, src[:0], dst[:0])


def test_copy_of_parts_of_pages():
    """Views whose rows are runs at equal distances, and a cache kept [heads, pages, ...]."""
    x = torch.randn(4, 30, 8, 16, device="cuda")
    want = x.clone()
    want[:, 7], want[:, 9, 2:5] = x[:, 3], x[:, 4, 2:5]
    one = lambda i: torch.tensor([i], dtype=torch.int32, device="cuda")  # noqa: E731
    copy_pages(x.transpose(0, 1), one(3), one(7))
    copy_pages(x.transpose(0, 1)[:, :, 2:5], one(4), one(9))
    assert torch.equal(x, want)


def test_a_run_of_all_operators():
    """Two prompts, three beams each: written, forked, extended, attended, selected and forked again by parents, compacted in between;
    two layers.  Every step's attention is that of a cache that keeps each beam's keys and values apart."""
    from llama3_np_b200 import PagedCache, beam_reorder, beam_select
    G, H, D, V, K = 2, 8, 64, 50, 3
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    cache = PagedCache(layers=2, kv_heads=G, head_dim=D, pages=40, page_size=8)
    waste = [cache.open() for _ in range(2)]
    cache.extend(waste, [30, 9])                                             # so that the prompts' pages begin further up
    prompts, count = [cache.open(), cache.open()], [21, 8]
    view = cache.extend(prompts, count)
    own = [[], []]                                                           # per layer: [beam] -> (keys, values) [tokens, G, D]
    for layer in range(2):
        k, v = rand(2, 21, G, D), rand(2, 21, G, D)
        cache.write(layer, view, k, v)
        own[layer] = [(k[b, :count[b]], v[b, :count[b]]) for b in range(2) for _ in range(K)]
    for w in waste:
        cache.free(w)
    beams = [s if j == 0 else cache.fork(s) for s in prompts for j in range(K)]
    history = torch.zeros(2 * K, 12, dtype=torch.int32, device="cuda")
    scores = torch.zeros(2, K, device="cuda")
    for step in range(12):
        if step in (3, 7):
            cache.compact()
        view = cache.extend(beams)
        for layer in range(2):
            q, kn, vn = rand(2 * K, H, D), rand(2 * K, G, D), rand(2 * K, G, D)
            out = cache.attend(layer, view, q, kn, vn)
            for r in range(2 * K):
                own[layer][r] = tuple(torch.cat([x, n[r:r + 1]]) for x, n in zip(own[layer][r], (kn, vn)))
                kk, vv = (x.double().repeat_interleave(H // G, 1) for x in own[layer][r])
                w = torch.softmax(torch.einsum("hd,thd->ht", q[r].double(), kk) * D ** -0.5, -1)
                want = torch.einsum("ht,thd->hd", w, vv)
                room = 2.0 ** -8 * want.abs() + 2.0 ** -12 * torch.einsum("ht,thd->hd", w, vv.abs())
                assert bool(((out[r].double() - want).abs() <= room).all()), (step, layer, r)
        logits = torch.randn(2, K, V, generator=g, device="cuda")
        scores, tokens, parents, _ = beam_select(logits, scores)
        beam_reorder([history], parents)
        history[:, step] = tokens.reshape(-1)
        p = [b * K + x for b, row in enumerate(parents.tolist()) for x in row]
        old, beams = beams, [cache.fork(beams[x]) for x in p]
        for s in old:
            cache.free(s)
        own = [[layer[x] for x in p] for layer in own]
    for s in beams:
        cache.free(s)
    assert cache.free_pages == cache.pages


def test_autograd_sees_what_is_written():
    """A backward pass that saved a pool's old values raises, as behind torch's own writes; and the device of a cache is a certain one."""
    from llama3_np_b200 import PagedCache, beam_reorder
    cache = PagedCache(layers=1, kv_heads=2, head_dim=64, pages=4, page_size=8, dtype=torch.float32)
    assert cache.device == torch.device("cuda", torch.cuda.current_device())
    seqs = [cache.open(), cache.open()]
    new = torch.ones(2, 2, 64, device="cuda")
    idx = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    state = torch.zeros(2, 3, device="cuda")
    view = cache.extend(seqs)
    for write in (lambda: cache.write(0, view, new[:, None], new[:, None]), lambda: cache.attend(0, view, torch.ones(2, 4, 64, device="cuda"), new, new),
                  lambda: copy_pages(cache.k, idx[:1], idx[1:])):
        w = torch.ones((), device="cuda", requires_grad=True)
        loss = (w * cache.k[0]).sum()
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    before = state._version
    beam_reorder(state, idx[None].flip(1).contiguous())
    assert state._version > before
    with torch.inference_mode():
        beam_reorder(torch.zeros(2, 3, device="cuda"), idx[None])
