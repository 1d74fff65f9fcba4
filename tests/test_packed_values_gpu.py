"""GPU suite: attention of a packed step where rows could reach one another."""
import math

import pytest
import torch

from llama3_np_b200 import paged_chunk_attention
from test_paged_chunk_gpu import TYPES, check, formula, make, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim,heads,n", [(48, 2, 32), (128, 4, 16), (64, 2, 7)])
@pytest.mark.parametrize("lengths", [[0, None], [5, None, -1], [None, 0, None, 0, 0]])
def test_requests_without_keys_between_others(kind, dim, heads, n, lengths):
    """A thread block that has rows without any key ahead of rows that see some: their queries lie in the same place."""
    requests = 900
    q, k, v, table, lens, starts = make(1, TYPES[kind], heads, 1, dim, 16, [(20, n)] * requests)
    for i, length in enumerate(lengths):
        if length is not None:
            lens[i::len(lengths)] = length
    got = check(q, k, v, table, lens, starts)
    for _ in range(3):
        assert torch.equal(paged_chunk_attention(q, k, v, table, lens, starts, out=torch.full_like(q, 3.0)), got)


def _place(table, b, p):
    return int(table[b, p // 16]), p % 16


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("sign", [1, -1])
def test_hidden_values_as_large_as_the_type_has_them(kind, dim, sign):
    """Later tokens, keys of every residue modulo 8 among them: the rows ahead of them do not change."""
    q, k, v, table, lens, starts = make(5, TYPES[kind], 8, 2, dim, 16, [(40, 100), (3000, 50), (0, 300)])
    want = formula(q, k, v, table, lens, starts)
    for b, first, last in ((0, 90, 140), (1, 3030, 3050), (2, 130, 300)):
        for p in range(first, last):
            page, at = _place(table, b, p)
            v[page, :, at] = sign * torch.finfo(TYPES[kind]).max
    got, lse = paged_chunk_attention(q, k, v, table, lens, starts, return_lse=True)
    keep = torch.cat([torch.arange(50), torch.arange(100, 130), torch.arange(150, 280)]).cuda()
    near(got[keep], lse[keep], [x[keep] for x in want])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("large", [1e30, None])
def test_keys_of_no_weight_under_large_values(kind, large):
    """A score of -infinity is no weight, however large the value, whichever key of a block has it."""
    q, k, v, table, lens, starts = make(6, TYPES[kind], 4, 2, 64, 16, [(700, 40), (0, 200)])
    large = min(large or torch.finfo(TYPES[kind]).max, torch.finfo(TYPES[kind]).max)
    q[..., 3] = q[..., 3].abs() + 0.01
    places = [_place(table, b, p) for b, first in ((0, 300), (1, 17)) for p in range(first, first + 11)]
    for page, at in places:
        v[page, :, at] = 0.0
    _, lse0, tol, tol_lse = formula(q, k, v, table, lens, starts)   # the bounds of finite keys: without the eleven, weights are e^(lse0 - lse) times as large
    for page, at in places:
        k[page, :, at, 3] = -math.inf
    out, lse, _, _ = formula(q, k, v, table, lens, starts)          # weights of 0: their values have no part in it
    seen = lse.isfinite()
    tol = torch.where(seen[..., None], tol * (lse0 - lse).exp()[..., None], tol)
    for page, at in places:
        v[page, :, at] = large
    got, lse_got = paged_chunk_attention(q, k, v, table, lens, starts, return_lse=True)
    near(got, lse_got, (out, lse, tol, tol_lse))
    assert bool(tol.isfinite().all())
