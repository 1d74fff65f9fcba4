"""GPU suite: beam selection among rows that begin at different places of 16 bytes."""
import pytest
import torch

from llama3_np_b200 import beam_select

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def best_of_equal_rows(row, K, n):
    """The n best (token, beam) of K beams with this row of logits and one score: by logit, then beam, then token; the sums play no part."""
    value, token = row.double().cpu().sort(descending=True, stable=True)
    res, at = [], 0
    while len(res) < n and at < len(value):
        same = token[at:][value[at:] == value[at]].tolist()  # sorted, and all equal ones
        res += [(t, k) for k in range(K) for t in same]
        at += len(same)
    return res[:n]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V", [257, 1001, 2049, 5003, 50257])
@pytest.mark.parametrize("K,n", [(2, 16), (5, 32), (9, 5)])
def test_equal_rows_at_any_address(kind, V, K, n):
    """Beams with the same logits and score: equal candidates come by beam, then token, wherever a row begins in memory."""
    g = torch.Generator(device="cuda").manual_seed(V * 10 + K)
    rows = (torch.randn(8, V, generator=g, device="cuda") * 3).to(TYPES[kind])
    want = [best_of_equal_rows(r, K, n) for r in rows]
    scores = torch.full((8, K), -3.25, device="cuda")
    wide = torch.zeros(8, K, V + 13, dtype=TYPES[kind], device="cuda")
    for first in [None, 0, 1, 3, 6]:
        if first is None:
            x = rows[:, None].expand(8, K, V).contiguous()
        else:
            x = wide[:, :, first:first + V]
            x.copy_(rows[:, None].expand(8, K, V))
        got, tokens, parents, _ = beam_select(x, scores, n)
        for b in range(8):
            assert list(zip(tokens[b].tolist(), parents[b].tolist())) == want[b], (first, b)
            same = {}
            for s, t in zip(got[b].tolist(), tokens[b].tolist()):
                assert same.setdefault(t, s) == s


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V", [1, 3, 17, 511, 513, 1030, 4097, 30001])
@pytest.mark.parametrize("n", [1, 33, 64])
@pytest.mark.parametrize("values", ["random", "few", "rare"])
def test_results_hang_on_no_address(kind, V, n, values):
    """The same logits at every phase of 16 bytes, with steps between rows that change it and steps that do not: bit for bit the same results."""
    g = torch.Generator(device="cuda").manual_seed(V + n)
    B, K = 3, 3
    x = torch.randn(B, K, V, generator=g, device="cuda") * 4
    if values == "few":
        x = x.round()                    # many equal ones
    elif values == "rare":
        x[torch.rand(x.shape, generator=g, device="cuda") < 0.97] = -torch.inf
    x = x.to(TYPES[kind])
    scores = torch.randn(B, K, generator=g, device="cuda")
    wide = -(-V // 8) * 8
    base = torch.zeros(B, K, wide, dtype=TYPES[kind], device="cuda")[:, :, :V]
    base.copy_(x)
    want = beam_select(base, scores, n, eos_id=0)
    for step, first in [(wide + 8, f) for f in range(8)] + [(V + 3, f) for f in range(3)] + [(V, 0)]:
        y = torch.full((B, K, step), 50.0, dtype=TYPES[kind], device="cuda")[:, :, first:first + V]  # what lies beside a row is larger
        y.copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(beam_select(y, scores, n, eos_id=0), want)), (step, first)
