"""CPU suite: results of a packed step's operators that would lie over what is read or written beside them are refused."""
import pytest
import torch

from llama3_np_b200 import paged_chunk_attention, paged_extend, paged_rotary_write


def _pools(dtype=torch.float32):
    both = torch.zeros(2, 5, 2, 16, 64, dtype=dtype)
    return both[0], both[1]


def _chunk(q, k, v, **kw):
    return paged_chunk_attention(q, k, v, torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which,at", [(0, 0), (1, 0), (0, 5 * 2 * 16 * 64 - 64), (1, 5 * 2 * 16 * 64 - 64)])
def test_attention_into_the_pools(dtype, which, at):
    k, v = _pools(dtype)
    q = torch.zeros(1, 2, 64, dtype=dtype)
    whole = torch.zeros(5 * 2 * 16 * 64 + 4096, dtype=dtype)
    pool = whole[:5 * 2 * 16 * 64].view(5, 2, 16, 64)
    with pytest.raises(ValueError, match="shares memory"):
        _chunk(q, *((pool, v) if which == 0 else (k, pool)), out=whole[at:at + 128].view(1, 2, 64))
    with pytest.raises(ValueError, match="CUDA device"):   # right behind them
        _chunk(q, *((pool, v) if which == 0 else (k, pool)), out=whole[5 * 2 * 16 * 64:][:128].view(1, 2, 64))


def test_attention_into_its_table_lengths_or_starts():
    k, v = _pools()
    q, words = torch.zeros(1, 2, 64), torch.zeros(1024, dtype=torch.int32)
    a = dict(page_table=torch.zeros(3, 4, dtype=torch.int32), lengths=torch.zeros(3, dtype=torch.int32), starts=torch.zeros(4, dtype=torch.int32))
    for name, size in (("page_table", (3, 4)), ("lengths", (3,)), ("starts", (4,))):
        own = words[100:][:a[name].numel()].view(size)
        with pytest.raises(ValueError, match="shares memory"):
            paged_chunk_attention(q, k, v, **{**a, name: own}, out=words.view(torch.float32)[:128].view(1, 2, 64))


@pytest.mark.parametrize("in_place", [False, True])
def test_turned_queries_into_the_pools(in_place):
    k, v = _pools()
    a = dict(k=torch.zeros(7, 2, 64), v=torch.zeros(7, 2, 64), positions=torch.zeros(7, dtype=torch.int32), slots=torch.zeros(7, dtype=torch.int64), k_pages=k, v_pages=v,
             frequencies=torch.zeros(32, dtype=torch.float64))
    for pool in (k, v):
        inside = pool.flatten()[128:128 + 7 * 4 * 64].view(7, 4, 64)
        with pytest.raises(ValueError, match="shares memory"):
            paged_rotary_write(inside if in_place else torch.zeros(7, 4, 64), **a, out=inside)


@pytest.mark.parametrize("name,size", [("lengths", 3), ("counts", 3), ("free_pages", 5)])
def test_pages_into_what_says_where_they_go(name, size):
    words = torch.zeros(64, dtype=torch.int32)
    a = dict(page_table=words[:12].view(3, 4), lengths=torch.zeros(3, dtype=torch.int32), counts=torch.zeros(3, dtype=torch.int32), free_pages=torch.zeros(5, dtype=torch.int32),
             page_size=16, tokens=7)
    with pytest.raises(ValueError, match="shares memory"):
        paged_extend(**{**a, name: words[11:11 + size]})
    with pytest.raises(ValueError, match="CUDA device"):
        paged_extend(**{**a, name: words[12:12 + size]})
