"""GPU suite: attention of a packed step where rows could reach one another."""
import pytest
import torch

from llama3_np_b200 import paged_chunk_attention
from test_paged_chunk_gpu import TYPES, check, make

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
