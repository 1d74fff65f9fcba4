"""GPU suite: attention of a packed step's rows over a cache in pages, against its formula in 64 bits."""
import ctypes as C
import math
import threading

import pytest
import torch

from llama3_np_b200 import _cabi, paged_attention, paged_chunk_attention

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(seed, dtype, heads, kv_heads, dim, page, requests, max_pages=None, spare=2, garbage=None, layout="heads", rest=0):
    """Queries of (tokens before, new ones) requests and `rest` rows of none, pools, a table of pages in random order, lengths and starts; places
    that no length reaches hold `garbage`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = [w + n for w, n in requests]
    need = [-(-n // page) for n in lens]
    total, wide = sum(need) + spare, max(need + [1]) if max_pages is None else max_pages
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
    starts = torch.tensor([0] + [n for _, n in requests]).cumsum(0).to(torch.int32)
    q = torch.randn(int(starts[-1]) + rest, heads, dim, generator=g, device="cuda").to(dtype)
    return q, k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), starts.cuda()


def formula(q, k, v, table, lens, starts, scale=None):
    """(out, lse, error bounds of both ahead of the last rounding) in 64 bits, request by request."""
    T, H, D = q.shape
    G, page = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device="cuda")
    tol = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    tol_lse = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    rows, first = table.cpu(), starts.tolist()
    part = 0.0 if k.dtype == torch.float32 else torch.finfo(k.dtype).eps / 2     # 16-bit weights
    for b in range(len(lens)):
        s0, n = first[b], first[b + 1] - first[b]
        total = max(int(lens[b]), 0)
        if n == 0:
            continue
        pos = [j for j in range(min(total, table.shape[1] * page)) if 0 <= int(rows[b, j // page]) < k.shape[0]]
        if not pos:
            continue
        ids = torch.tensor([int(rows[b, j // page]) for j in pos], device="cuda")
        off = torch.tensor([j % page for j in pos], device="cuda")
        at = total - n + torch.arange(n, device="cuda")
        hidden = (torch.tensor(pos, device="cuda") > at[:, None])[:, None]
        none = hidden.all(-1)
        for g in range(G):
            hs = slice(g * (H // G), (g + 1) * (H // G))
            kk, vv, qq = k[ids, g, off].double(), v[ids, g, off].double(), q[s0:s0 + n, hs].double()
            s = torch.einsum("thd,kd->thk", qq, kk) * scale
            s = s.masked_fill(hidden, -math.inf)
            w = torch.softmax(s, -1)
            w = torch.where(none[..., None], torch.zeros_like(w), w).masked_fill(hidden, 0)
            def sums(x):  # a value that a row does not see has no part in it
                clean = torch.einsum("thk,kd->thd", w, torch.where(x.isfinite(), x, 0))
                odd = ~x.isfinite().all(-1)
                if odd.any():
                    see = (~hidden[:, :, odd]).to(x.dtype)
                    for j, value in enumerate(x[odd]):
                        clean = torch.where((see[..., j] > 0)[..., None] & ~value.isfinite(), clean + value, clean)
                return clean
            out[s0:s0 + n, hs] = torch.where(none[..., None], torch.zeros((), dtype=torch.float64, device="cuda"), sums(vv))
            lse[s0:s0 + n, hs] = torch.logsumexp(s, -1)
            # scores: D products summed in fp32 (tensor cores may cut instead of round: a step of 2^-22 each); exponentials 2^-21 and what the
            # argument's last bit makes of it; the weights' rounding; sums of the keys, 16 at a time, and the join
            es = (qq.abs() @ kk.abs().T).amax(-1) * abs(scale) * (D + 2) * 2.0 ** -22
            big = torch.where(hidden, torch.zeros_like(s), s).abs().amax(-1)
            delta = 2 * (es + big * 2.0 ** -22 + 2.0 ** -20) + part + (len(pos) / 16 + 64) * 2.0 ** -22
            finite = torch.where(vv.isfinite(), vv.abs(), 0)
            tol[s0:s0 + n, hs] = delta[..., None] * torch.einsum("thk,kd->thd", w.nan_to_num(0), finite)
            tol_lse[s0:s0 + n, hs] = delta - part
            if k.dtype == torch.float16:  # the largest weight is scaled to 2^12 at least, and fp16's smallest number is 2^-24: half of it is 2^-37 of the largest
                tol[s0:s0 + n, hs] += len(pos) * 2.0 ** -37 * finite.amax()
    return out, lse, tol, tol_lse


def near(got, lse, want):
    """Within the bounds; equal where not finite."""
    want, want_lse, tol, tol_lse = want
    dtype = got.dtype
    err = (got.double() - want).abs()
    bound = tol + want.abs() * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == torch.float16 else 0)
    fine = want.isfinite()
    assert torch.equal(got.isfinite(), fine) and torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.double()[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    assert bool((err <= bound)[fine].all()), f"worst {float((err / bound.clamp(min=1e-30))[fine].max()):.3f} of the bound"
    fine = want_lse.isfinite()
    assert torch.equal(lse.isfinite(), fine) and torch.equal(lse.isnan(), want_lse.isnan())
    lse_tol = tol_lse + want_lse.abs() * 2.0 ** -23
    assert bool(((lse.double() - want_lse).abs() <= lse_tol)[fine].all())


def check(q, k, v, table, lens, starts, scale=None, **kw):
    got, lse = paged_chunk_attention(q, k, v, table, lens, starts, scale=scale, return_lse=True, **kw)
    assert got.dtype == q.dtype and got.shape == q.shape and lse.shape == q.shape[:2]
    near(got, lse, formula(q, k, v, table, lens, starts, scale))
    return got


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(6, 6), (8, 1), (6, 2), (28, 4), (20, 1)])
def test_shapes(kind, dim, heads, kv_heads):
    check(*make(dim + heads, TYPES[kind], heads, kv_heads, dim, 16, [(0, 37), (100, 1), (0, 0), (5, 130), (300, 20), (0, 1), (15, 1)], garbage=math.nan))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 64, 256])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_pages_and_layouts(kind, page, layout):
    check(*make(page, TYPES[kind], 8, 2, 64, page, [(0, page), (page, 1), (100, 33), (7, 200), (0, 300)], garbage=math.inf, layout=layout))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [48, 64, 128])
@pytest.mark.parametrize("requests", [[(20000, 3)], [(9001, 200)], [(0, 2500)], [(3000, 1), (0, 700), (5000, 5)], [(700, 1)] * 40, [(10, 5)] * 300, [(3, 1)] * 1500,
                                      [(0, 129), (4000, 64), (0, 1), (128, 128), (127, 1)]])
def test_split_and_joined(kind, dim, requests):
    """From one request over all SMs to more requests than threads."""
    args = make(len(requests), TYPES[kind], 4, 2, dim, 16, requests)
    got = check(*args)
    assert torch.equal(got, paged_chunk_attention(*args)), "results change from run to run"
    out = check(*args, out=torch.empty_like(got))     # few rows go another way where the result is made by the call
    assert torch.equal(out, paged_chunk_attention(*args, out=torch.empty_like(got)))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim,heads,kv_heads", [(16, 4, 4), (48, 6, 2), (128, 32, 8)])
@pytest.mark.parametrize("requests", [[(1500, 5)], [(0, 1)], [(0, 0), (7, 2), (0, 0), (300, 1), (0, 3), (40, 0)], [(3, 1)] * 16, [(100, 0)] * 50 + [(90, 9)] + [(1, 0)] * 50])
@pytest.mark.parametrize("rest", [0, 4])
def test_few_rows(kind, dim, heads, kv_heads, requests, rest):
    args = make(len(requests), TYPES[kind], heads, kv_heads, dim, 16, requests, garbage=math.nan, rest=rest)
    got, n = check(*args), int(args[-1][-1])
    assert not got[n:].any()
    out = torch.full_like(got, 7.0)
    paged_chunk_attention(*args, out=out)
    assert bool((out[n:] == 7).all())
    near(out[:n], paged_chunk_attention(*args, return_lse=True)[1][:n], [x[:n] for x in formula(*args)])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rest", [1, 200])
def test_rows_of_no_request(kind, rest):
    args = make(1, TYPES[kind], 8, 2, 64, 16, [(30, 20), (0, 0), (5, 7)], rest=rest)
    q, starts = args[0], args[-1]
    got = check(*args)
    n = int(starts[-1])
    assert not got[n:].any()
    out = torch.full_like(q, 7.0)
    again = paged_chunk_attention(*args, out=out)
    assert again is out and torch.equal(out[:n], got[:n]) and bool((out[n:] == 7).all())


def test_no_requests_and_no_rows():
    q, k, v, table, lens, starts = make(1, torch.bfloat16, 8, 2, 64, 16, [(30, 20)])
    out, lse = paged_chunk_attention(q, k, v, table[:0], lens[:0], starts[:1], return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    out, lse = paged_chunk_attention(q[:0], k, v, table, lens, starts, return_lse=True)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
    out = torch.full_like(q, 3.0)
    paged_chunk_attention(q, k, v, table, lens, torch.zeros_like(starts), out=out)
    assert bool((out == 3).all())


@pytest.mark.parametrize("kind", list(TYPES))
def test_lengths_below_the_rows_beyond_the_table_and_below_zero(kind):
    q, k, v, table, lens, starts = make(3, TYPES[kind], 4, 2, 64, 16, [(20, 30)] * 5)
    lens.copy_(torch.tensor([10, -5, 0, 200, 2 ** 31 - 1], dtype=torch.int32))   # rows at negative positions, and all tokens of the table
    got = check(q, k, v, table, lens, starts)
    assert not got[:20].any() and not got[30:90].any() and got[20:30].any()


@pytest.mark.parametrize("kind", list(TYPES))
def test_pages_that_are_not_there(kind):
    q, k, v, table, lens, starts = make(4, TYPES[kind], 6, 2, 48, 8, [(300, 40), (0, 60), (9, 9)])
    table[0, ::3] = -1
    table[0, 4] = 2 ** 30
    table[1] = k.shape[0]
    table[2, 0] = -7
    got = check(q, k, v, table, lens, starts)
    assert not got[40:100].any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_has_no_part(kind, dim, bad):
    """The later tokens' values and keys are no numbers: rows ahead of them do not change."""
    q, k, v, table, lens, starts = make(5, TYPES[kind], 8, 2, dim, 16, [(40, 100), (3000, 50)])
    want = formula(q, k, v, table, lens, starts)
    for b, p in ((0, 90), (1, 3030)):
        page, off = int(table[b, p // 16]), p % 16
        k[page, :, off] = bad
        v[page, :, off] = bad
    got, lse = paged_chunk_attention(q, k, v, table, lens, starts, return_lse=True)
    keep = torch.cat([torch.arange(50), torch.arange(100, 130)]).cuda()
    near(got[keep], lse[keep], [x[keep] for x in want])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(kind, bad):
    q, k, v, table, lens, starts = make(6, TYPES[kind], 4, 2, 64, 16, [(20, 60), (2000, 9)])
    for b, p in ((0, 45), (1, 700)):
        v[int(table[b, p // 16]), 1, p % 16, 3] = bad
    check(q, k, v, table, lens, starts)


def test_queries_and_keys_that_are_no_numbers():
    q, k, v, table, lens, starts = make(7, torch.bfloat16, 4, 2, 64, 16, [(20, 60)])
    q[5, 1, 3], q[6, 2, 0] = math.nan, math.inf
    k[int(table[0, 2]), 0, 3, 7] = math.nan      # token 35: position 15 of the rows
    got, lse = paged_chunk_attention(q, k, v, table, lens, starts, return_lse=True)
    nan = torch.zeros(60, 4, dtype=torch.bool, device="cuda")
    nan[5, 1] = nan[6, 2] = True
    nan[15:, :2] = True
    assert torch.equal(lse.isnan(), nan) and torch.equal(got.isnan().all(-1), nan) and torch.equal(got.isnan().any(-1), nan)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7, 12.0])
def test_scales(kind, scale):
    check(*make(8, TYPES[kind], 8, 2, 64, 16, [(500, 90), (0, 140)]), scale=scale)


@pytest.mark.parametrize("kind", list(TYPES))
def test_maxima_that_grow_along_the_keys(kind):
    """Every block's scores are far above the ones before: what was summed so far is scaled down each time."""
    q, k, v, table, lens, starts = make(9, TYPES[kind], 4, 2, 128, 16, [(1500, 70)])
    q.abs_()
    for j in range(1570):
        k[int(table[0, j // 16]), :, j % 16] = (j - 700) / 200
    check(q, k, v, table, lens, starts)


def test_many_small_weights_beside_a_large_one():
    """fp16: 30000 weights of 2^-20 of the largest make 3 % of the sum."""
    q, k, v, table, lens, starts = make(10, torch.float16, 2, 1, 64, 64, [(30000, 3)])
    q.zero_(), k.zero_()
    q[..., 0] = 1.0
    k[int(table[0, 100]), 0, 5, 0] = 20 * math.log(2) * 8
    v.abs_()
    check(q, k, v, table, lens, starts)


def test_strided_queries():
    _, k, v, table, lens, starts = make(11, torch.bfloat16, 8, 2, 64, 16, [(30, 50), (7, 1)])
    qkv = torch.randn(51, 12 * 64, device="cuda").bfloat16()
    q = qkv[:, :8 * 64].view(51, 8, 64)
    assert torch.equal(check(q, k, v, table, lens, starts), paged_chunk_attention(q.contiguous(), k, v, table, lens, starts))
    check(torch.randn(8, 51, 64, device="cuda").bfloat16().transpose(0, 1), k, v, table, lens, starts)
    check(torch.randn(51, 1, 64, device="cuda").bfloat16().expand(51, 8, 64), k, v, table, lens, starts)


@pytest.mark.parametrize("kind", list(TYPES))
def test_single_tokens_as_paged_attention_has_them(kind):
    q, k, v, table, lens, starts = make(12, TYPES[kind], 8, 2, 64, 16, [(n, 1) for n in (0, 15, 16, 900, 77, 3000)])
    a, la = paged_chunk_attention(q, k, v, table, lens, starts, return_lse=True)
    b, lb = paged_attention(q, k, v, table, lens, return_lse=True)
    eps = torch.finfo(TYPES[kind]).eps
    assert torch.allclose(a.float(), b.float(), rtol=2 * eps, atol=4 * eps) and torch.allclose(la, lb, rtol=1e-5, atol=1e-5)


def test_captured_with_other_lengths_and_on_another_stream():
    requests = [(200, 40), (0, 60), (33, 1)]
    q, k, v, table, lens, starts = make(13, torch.bfloat16, 8, 2, 128, 16, requests, max_pages=20, rest=99)
    out, out2 = torch.zeros_like(q), torch.zeros_like(q)
    paged_chunk_attention(q, k, v, table, lens, starts, out=out)
    graphs = []
    for o in (out, out2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            paged_chunk_attention(q, k, v, table, lens, starts, out=o)
        graphs.append(g)
    lens.copy_(torch.tensor([101, 100, 33], dtype=torch.int32))
    starts.copy_(torch.tensor([0, 100, 190, 191], dtype=torch.int32))
    out.fill_(5.0), out2.fill_(5.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
        eager = paged_chunk_attention(q, k, v, table, lens, starts)
    torch.cuda.synchronize()
    want = check(q, k, v, table, lens, starts)
    assert torch.equal(out[:191], want[:191]) and bool((out[191:] == 5).all()) and torch.equal(out, out2) and torch.equal(eager, want)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_pools_beyond_32_bits(kind):
    """A pool of more than 2^31 values, its last pages in use, and of 2^32 bytes."""
    dtype = TYPES[kind]
    pages = (1 << 31) // (2 * 16 * 64) + 300
    k = torch.empty(pages, 2, 16, 64, dtype=dtype, device="cuda")
    v = torch.empty(pages, 2, 16, 64, dtype=dtype, device="cuda")
    ids = torch.cat([torch.arange(pages - 20, pages), torch.arange(5), torch.arange(pages // 2, pages // 2 + 10)]).int()
    for p in (k, v):
        p[ids.long().cuda()] = torch.randn(35, 2, 16, 64, device="cuda").to(dtype)
    table = ids[torch.randperm(35, generator=torch.Generator().manual_seed(1))][None].cuda()
    q = torch.randn(90, 4, 64, device="cuda").to(dtype)
    check(q, k, v, table, torch.tensor([550], dtype=torch.int32, device="cuda"), torch.tensor([0, 90], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("requests", [[(60, 9), (0, 0), (3, 1)], [(30, 70), (0, 0), (5, 17)]])
def test_rows_ahead_of_the_first_request(kind, requests):
    """Rows ahead of starts[0] belong to no request, either: 0, or as they are in `out`; what is made here is always set."""
    ahead = 3
    args = list(make(2, TYPES[kind], 8, 2, 64, 16, requests, rest=ahead + 2))
    args[-1] = args[-1] + ahead
    got = check(*args)
    n = int(args[-1][-1])
    out = torch.full_like(args[0], 7.0)
    torch.full((1 << 16,), 5.0, device="cuda")   # what lse's memory may hold
    again, lse = paged_chunk_attention(*args, out=out, return_lse=True)
    none = torch.ones(len(out), dtype=torch.bool, device="cuda")
    none[ahead:n] = False
    assert torch.allclose(again[~none].float(), got[~none].float(), rtol=2e-2, atol=2e-2)
    assert bool((again[none] == 7).all()) and bool((lse[none] == -math.inf).all()) and bool(lse[~none].isfinite().all())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("how", ["pages of both", "one behind the other", "values first", "the same", "rows of both"])
@pytest.mark.parametrize("page", [4, 16, 256])
def test_pools_in_one_piece_of_memory(kind, how, page):
    q, k, v, table, lens, starts = make(3, TYPES[kind], 8, 2, 64, page, [(300, 40), (0, 170), (77, 1)], garbage=math.nan)
    if how == "pages of both":
        k, v = torch.stack([k, v], 1).unbind(1)
    elif how == "one behind the other":
        k, v = torch.stack([k, v]).unbind(0)
    elif how == "values first":
        v, k = torch.stack([v, k]).unbind(0)
    elif how == "rows of both":
        v, k = torch.cat([v, k], -1).split(64, -1)
    else:
        v = k
    check(q, k, v, table, lens, starts)


@pytest.mark.parametrize("kind", list(TYPES))
def test_a_table_without_columns(kind):
    q, k, v, table, lens, starts = make(4, TYPES[kind], 8, 2, 64, 16, [(30, 20), (5, 7)])
    out, lse = paged_chunk_attention(q, k, v, table[:, :0], lens, starts, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 64, 128])
def test_results_on_16_bytes(kind, dim):
    args = make(5, TYPES[kind], 8, 2, dim, 16, [(300, 140), (5, 7)])
    want = check(*args)
    out = torch.empty(want.numel() + 8, dtype=want.dtype, device="cuda")[8:].view_as(want)
    assert torch.equal(paged_chunk_attention(*args, out=out), want)


@pytest.mark.parametrize("kind", list(TYPES))
def test_a_workspace_on_16_bytes(kind):
    """As the C interface asks for it, and no byte around it is written."""
    q, k, v, table, lens, starts = make(6, TYPES[kind], 8, 2, 64, 16, [(5000, 40), (0, 170)])
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    code = {"f32": _cabi.DTYPE_F32, "bf16": _cabi.DTYPE_BF16, "f16": _cabi.DTYPE_F16}[kind]
    need = C.c_int64()
    lib = _cabi.lib()
    assert lib.l3_paged_chunk_workspace(0, len(q), 8, 2, 64, code, C.byref(need)) == 0
    room = torch.full((need.value + 256,), 77, dtype=torch.uint8, device="cuda")
    begin = 16 if room.data_ptr() % 32 == 0 else 0
    a = _cabi.L3PagedChunk(device=0, batch=2, tokens=len(q), heads=8, kv_heads=2, head_dim=64, pages=len(k), page_size=16, max_pages=table.shape[1], dtype=code,
                           clear_rest=1, scale=0.125, stream=torch.cuda.current_stream().cuda_stream, q=q.data_ptr(), q_token_stride=512, q_head_stride=64,
                           k=_cabi.L3PagePool(k.data_ptr(), *k.stride()[:3]), v=_cabi.L3PagePool(v.data_ptr(), *v.stride()[:3]), table=table.data_ptr(),
                           table_stride=table.stride(0), lengths=lens.data_ptr(), starts=starts.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
                           workspace=room.data_ptr() + begin, workspace_bytes=need.value)
    assert lib.l3_paged_chunk_attention(C.byref(a)) == 0
    near(out, lse, formula(q, k, v, table, lens, starts))
    assert bool((room[:begin] == 77).all()) and bool((room[begin + need.value:] == 77).all())


def test_several_streams_and_threads_at_once():
    cases = [make(20 + i, dtype, 8, 2, dim, 16, requests) for i, (dtype, dim, requests) in enumerate([
        (torch.bfloat16, 128, [(900, 300), (0, 500)]), (torch.float16, 64, [(3000, 30)] * 4), (torch.float32, 48, [(100, 90)] * 6), (torch.bfloat16, 64, [(40, 5)])])]
    want = [paged_chunk_attention(*c) for c in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got[i].append(paged_chunk_attention(*cases[i]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for w, all_of in zip(want, got):
        assert len(all_of) == 50 and all(torch.equal(w, x) for x in all_of)
