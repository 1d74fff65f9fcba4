"""GPU suite: attention over a cache in pages at values that are infinite, and at queries of any size."""
import math

import pytest
import torch

from llama3_np_b200 import paged_attention

pytestmark = pytest.mark.gpu
HALVES = {"bf16": torch.bfloat16, "f16": torch.float16}


def make(seed, dtype, heads, kv_heads, dim, lens, max_pages, page=16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lens), max_pages or max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    k = torch.randn(at, kv_heads, page, dim, generator=g, device="cuda").to(dtype)
    v = torch.randn(at, kv_heads, page, dim, generator=g, device="cuda").to(dtype)
    q = torch.randn(len(lens), heads, dim, generator=g, device="cuda")
    return q, k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def definition(q, k, v, table, lens, scale):
    """(out, lse, bounds of their errors ahead of the last rounding) in 64 bits.  A key whose score is -inf has no weight."""
    B, H, D = q.shape
    G, page = k.shape[1], k.shape[2]
    out, tol = torch.zeros(2, B, H, D, dtype=torch.float64, device="cuda")
    lse, tol_lse = torch.zeros(2, B, H, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens.tolist()):
        ids = table[b, :-(-n // page)].long()
        for h in range(H):
            g = h // (H // G)
            kk, vv, qq = k[ids, g].reshape(-1, D)[:n].double(), v[ids, g].reshape(-1, D)[:n].double(), q[b, h].double()
            s = (kk * qq).sum(-1) * scale
            if bool(s.isnan().any()) or bool((s == math.inf).any()):
                out[b, h], lse[b, h] = math.nan, s.logsumexp(-1)
                continue
            seen = s > -math.inf
            s, kk, vv = s[seen], kk[seen], vv[seen]
            w = torch.softmax(s, -1)
            out[b, h], lse[b, h] = (w[:, None] * vv).sum(0), torch.logsumexp(s, -1)
            # scores: D products summed in fp32, a step of 2^-22 each; an fp32 query's two parts: 2^-16 (bf16) and 2^-21 (fp16) of a value, or (fp16)
            # 2^-39 of the row's largest; weights: two parts of 8 bits and a sign (bf16, 2^-16), of 11 (fp16, 2^-21) or 2^-36 of the largest weight
            bf, two = k.dtype == torch.bfloat16, q.dtype != k.dtype
            parts = 0.0 if not two else 2.0 ** -16 if bf else 2.0 ** -21
            es = ((qq.abs() * kk.abs()).sum(-1) * ((D + 2) * 2.0 ** -22 + parts) + (0 if bf or not two else qq.abs().max() * kk.abs().sum(-1) * 2.0 ** -39)).max() * abs(scale)
            delta = 2 * (es + s.abs().max() * 2.0 ** -22 + 2.0 ** -20 + (2.0 ** -16 if bf else 2.0 ** -21)) + (n / 16 + 64) * 2.0 ** -22
            fine = vv.abs().nan_to_num(0, 0, 0)
            tol[b, h] = delta * (w[:, None] * fine).sum(0) + (0 if bf else 2.0 ** -36 * w.max() * fine.sum(0))
            tol_lse[b, h] = delta
    return out, lse, tol, tol_lse


def check(q, k, v, table, lens, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    got, lse = paged_attention(q, k, v, table, lens, scale=scale, return_lse=True)
    want, want_lse, tol, tol_lse = definition(q, k, v, table, lens, scale)
    x, fine = got.double(), want.isfinite()
    assert torch.equal(x.isnan(), want.isnan()) and torch.equal(x[want.isinf()], want[want.isinf()])
    bound = tol + want.abs() * torch.finfo(q.dtype).eps / 2 + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    assert bool(((x - want).abs()[fine] <= bound[fine]).all())
    some = want_lse.isfinite()
    assert bool(((lse.double() - want_lse).abs()[some] <= (tol_lse + want_lse.abs() * 2.0 ** -23)[some]).all())
    return got


PLANS = [([37, 1, 150, 17], None), ([700], None), ([300, 5, 64], 4000)]   # a block, a cluster an item; all warps share all items


@pytest.mark.parametrize("kind", list(HALVES))
@pytest.mark.parametrize("dim", [16, 48, 64, 96, 128])
@pytest.mark.parametrize("two_parts", [False, True])
@pytest.mark.parametrize("lens,wide", PLANS)
def test_infinite_values(kind, dim, two_parts, lens, wide):
    """A weight is positive, however its rounding falls: an infinite value makes its dimension infinite, of two signs or NaN it makes it NaN."""
    for seed in range(4):
        q, k, v, table, n = make(seed + dim, HALVES[kind], 6, 3, dim, lens, wide)
        q = q if two_parts else q.to(k.dtype)
        for b, m in enumerate(lens):
            at = lambda j: (table[b, j // 16].long(), slice(None), j % 16)
            v[at(m // 2)][:, 0], v[at(m - 1)][:, 1] = math.inf, -math.inf
            v[at(0)][:, 2], v[at(m - 1)][:, 2] = math.inf, -math.inf   # (of one token: -inf alone)
            v[at(m // 3)][:, 3] = math.nan
            v[at(m // 2)][:, 4:8], v[at(m // 3)][:, 4:8] = math.inf, math.inf
        check(q, k, v, table, n)


@pytest.mark.parametrize("kind", list(HALVES))
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("two_parts", [False, True])
@pytest.mark.parametrize("lens,wide", PLANS)
def test_infinite_keys(kind, dim, two_parts, lens, wide):
    """A score of -inf is no weight, one of +inf makes the query's result NaN; the other queries of the kv head are not touched."""
    for seed in range(4):
        q, k, v, table, n = make(seed + dim, HALVES[kind], 6, 3, dim, lens, wide)
        q[:, ::2, 3], q[:, 1::2, 3] = q[:, ::2, 3].abs() + 0.01, -q[:, 1::2, 3].abs() - 0.01
        q = q if two_parts else q.to(k.dtype)
        for b, m in enumerate(lens):
            if m > 1:
                k[table[b, (m // 2) // 16].long(), :, (m // 2) % 16, 3] = -math.inf  # -inf for even heads, +inf for odd ones
        got = check(q, k, v, table, n)
        assert got[:, ::2].isfinite().all()


def test_infinite_value_of_a_small_weight():
    """fp16: a weight that 16 bits have no number for is still a weight."""
    q, k, v, table, n = make(1, torch.float16, 2, 2, 64, [200], None)
    k.mul_(0.01)
    k[:, :, :, 0] = 0
    q[:, :, 0] = 8
    k[table[0, 2].long(), :, 3, 0] = 30      # scores 30 and about 0: weights e^-30 of the largest
    v[table[0, 5].long(), :, 1, 7] = math.inf
    check(q.half(), k, v, table, n)
    check(q, k, v, table, n)


def test_infinite_key_under_a_small_query_value():
    q, k, v, table, n = make(2, torch.float16, 4, 2, 32, [90], None)
    q[:, :, 5] = 2.0 ** -60
    k[table[0, 1].long(), :, 7, 5] = -math.inf
    check(q, k, v, table, n)


@pytest.mark.parametrize("kind", list(HALVES))
@pytest.mark.parametrize("dim", [48, 64, 128])
@pytest.mark.parametrize("lens,wide", PLANS)
def test_fp32_queries_of_any_size(kind, dim, lens, wide):
    """Queries 2^e times as large under a scale 2^-e times as large are the same queries, bit for bit."""
    q, k, v, table, n = make(7, HALVES[kind], 6, 3, dim, lens, wide)
    q[:, 1] *= 2.0 ** -12    # every head by itself
    q[:, 2] *= 2.0 ** -12
    q[:, 2, 0] = 1.0
    base = check(q, k, v, table, n, scale=0.25)
    for e in (-60, -24, -14, -3, 11, 17, 60):
        assert torch.equal(check(q * 2.0 ** e, k, v, table, n, scale=0.25 * 2.0 ** -e), base)


def test_largest_fp32_queries():
    q, k, v, table, n = make(8, torch.bfloat16, 4, 2, 64, [100, 3], None)
    q = torch.where(q > 0, 3.4e38, -3.4e38) * (torch.arange(64, device="cuda") % 5 == 0)
    check(q, k, v, table, n, scale=1.2e-38)


@pytest.mark.parametrize("kind", list(HALVES))
@pytest.mark.parametrize("two_parts", [False, True])
@pytest.mark.parametrize("ahead", [4, 9, 13, 17, 25, 40])
@pytest.mark.parametrize("wide", [None, 4000])
def test_many_small_weights_beside_a_large_one(kind, two_parts, ahead, wide):
    """One key whose score is `ahead` above some 3000 others': weights that 16 bits hold with all their bits, a few of them, and none."""
    q, k, v, table, n = make(ahead, HALVES[kind], 4, 2, 64, [3001], wide)
    q[:, :, 0], k[:, :, :, 0] = 8.0, 0.0
    k[table[0, 77].long(), :, 5, 0] = float(ahead)
    k[..., 1:] *= 0.25
    v[table[0, 77].long(), :, 5] = 0.0   # the small ones are what is left
    check(q if two_parts else q.to(k.dtype), k, v, table, n)


@pytest.mark.parametrize("two_parts", [False, True])
def test_large_keys(two_parts):
    """bf16 keys as large as fp32's under a scale that makes their scores ordinary ones: no product of theirs and a query's is infinite."""
    q, k, v, table, n = make(9, torch.bfloat16, 4, 2, 64, [100, 3, 700], None)
    k *= torch.where(torch.arange(64, device="cuda") % 9 == 0, 1e37, 1e30)
    q = q.clamp(-3, 3)
    check(q if two_parts else q.bfloat16(), k, v, table, n, scale=2e-38)
    if two_parts:
        check(q * 2.0 ** -70, k, v, table, n, scale=2e-38 * 2.0 ** 70)
