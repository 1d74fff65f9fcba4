"""GPU suite: beam search's selection and reordering, against their definitions."""
import math

import pytest
import torch

from llama3_np_b200 import beam_reorder, beam_select

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def formula(logits, scores, best, done=None, eos=None):
    """By sorting all candidates in 64 bits: [(score, beam, token)] per sequence, at most `best`."""
    B, K, V = logits.shape
    out = []
    for b in range(B):
        cand = []
        for k in range(K):
            s = float(scores[b, k])
            if done is not None and bool(done[b, k]):
                cand.append((s, k, eos))
                continue
            p = s + torch.log_softmax(logits[b, k].double(), -1).cpu()
            keep = torch.sort(p, descending=True, stable=True)
            cand += [(float(x), k, int(t)) for x, t in zip(keep.values[:best + 1], keep.indices[:best + 1])]
        cand = [c for c in cand if math.isfinite(c[0])]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        out.append(cand)
    return out


def check(logits, scores, best, done=None, eos=None):
    s, t, p, d = beam_select(logits, scores, best, done=done, eos_id=eos)
    assert s.shape == t.shape == p.shape == d.shape == (logits.shape[0], best)
    for b, cand in enumerate(formula(logits, scores, best, done, eos)):
        # candidates of different beams that lie closer than what the sums of exponentials can be off by would say nothing
        for x, y in zip(cand[:best], cand[1:]):
            assert x[1] == y[1] or x[0] == y[0] or x[0] - y[0] > 2.0 ** -19, "pick another seed"
        for i in range(best):
            if i >= len(cand):
                assert float(s[b, i]) == -math.inf and int(p[b, i]) == 0 and int(t[b, i]) == (0 if eos is None else eos) and bool(d[b, i])
                continue
            x, k, v = cand[i]
            assert (int(p[b, i]), int(t[b, i])) == (k, v), (b, i)
            # fp32 exponentials are off by 2^-21 relative, their sum and its logarithm by no more, and the score is rounded once
            assert abs(float(s[b, i]) - x) <= abs(x) * 2.0 ** -24 + 2.0 ** -20
            assert bool(d[b, i]) == ((done is not None and bool(done[b, k])) or (eos is not None and v == eos))


def make(seed, B, K, V, dtype, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, K, V, generator=g, device="cuda") * scale).to(dtype), -10 * torch.rand(B, K, generator=g, device="cuda")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("B,K,V,best", [(1, 1, 1, 1), (1, 4, 32000, 4), (3, 1, 7, 3), (2, 5, 1000, 10), (4, 2, 257, 64), (1, 64, 513, 64),
                                        (7, 3, 128256, 6), (2, 200, 50, 17), (40, 8, 4097, 8)])
def test_select(kind, B, K, V, best):
    logits, scores = make(B * 100 + K, B, K, V, TYPES[kind])
    check(logits, scores, best)


@pytest.mark.parametrize("V", [5, 300, 33000])
def test_finished_beams(V):
    logits, scores = make(V, 4, 4, V, torch.float32)
    done = torch.tensor([[0, 1, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0], [1, 0, 1, 1]], device="cuda").bool()
    logits[0, 1] = math.nan                    # a finished beam's logits are not looked at
    check(logits, scores, 4, done, 3)
    check(logits, scores, 6, done, 3)
    check(logits, scores, 4, done.to(torch.uint8), 0)
    check(logits[2:3], scores[2:3], 4, None, 2)


@pytest.mark.parametrize("V", [64, 5000, 40000])
@pytest.mark.parametrize("best", [1, 4, 64])
def test_equal_scores(V, best):
    """More equal values than there is room for: the lowest indices win, in order."""
    logits = torch.zeros(2, 2, V, device="cuda")
    scores = torch.tensor([[0.0, 0.0], [-1.0, -0.5]], device="cuda")
    s, t, p, _ = beam_select(logits, scores, best)
    assert t[0].tolist() == list(range(best)) and p[0].tolist() == [0] * best
    assert t[1].tolist() == list(range(best)) and p[1].tolist() == [1] * best
    logits[0, 1, V - 5:] = 1.0
    logits[:, :, 10] = -0.0                    # equal to 0
    check(logits, scores, min(best, 4))


def test_masked_tokens():
    logits, scores = make(3, 2, 3, 900, torch.float32)
    logits[0] = -math.inf
    logits[0, 0, 5], logits[0, 2, 800] = 1.0, 0.5          # two continuations are left
    logits[1, 0, :899] = -math.inf
    scores[1, 2] = -math.inf                               # no such beam
    check(logits, scores, 5)
    logits[1] = -math.inf
    check(logits, scores, 2, None, 7)
    low = torch.finfo(torch.float32).min
    logits[1] = low
    logits[1, 1, 3:9] = 0.0
    check(logits, scores, 3)


def test_values_that_are_not_numbers():
    logits, scores = make(4, 1, 3, 700, torch.float32)
    logits[0, 0, 9] = math.nan                             # such a row has no continuation, nor has one with +inf
    logits[0, 1, 30] = math.inf
    s, t, p, _ = beam_select(logits, scores, 4)
    assert p.tolist() == [[2] * 4]
    want = torch.topk(logits[0, 2], 4).indices
    assert t[0].tolist() == want.tolist()
    logits[0, 2, 0] = math.nan
    s, t, p, d = beam_select(logits, scores, 2)
    assert bool((s == -math.inf).all()) and d.all()


def test_strides_large_logits_and_streams():
    logits, scores = make(6, 3, 4, 3001, torch.float32)
    wide = torch.zeros(3, 5, 3003, device="cuda")
    wide[:, 1:, 1:3002] = logits * 40
    check(wide[:, 1:, 1:3002], scores, 4)
    want = beam_select(logits, scores, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = beam_select(logits, scores, 4)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = beam_select(logits, scores, 4)
    logits.neg_()
    g.replay()
    assert all(torch.equal(x, y) for x, y in zip(got, beam_select(logits, scores, 4)))
    assert beam_select(logits[:0], scores[:0])[0].shape == (0, 4)


# ---------------------------------------------------------------------------------------------------------- reordering
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (16, 128, 128)), (torch.int32, (511,)), (torch.bfloat16, (3, 7)), (torch.uint8, (13,)),
                                         (torch.bool, (64,)), (torch.float32, ())])
@pytest.mark.parametrize("B,K", [(1, 1), (3, 4), (2, 64), (1, 256), (5, 7)])
def test_reorder(dtype, shape, B, K):
    g = torch.Generator(device="cuda").manual_seed(K)
    x = [torch.randint(0, 2, (B * K,) + shape, generator=g, device="cuda").to(dtype) if dtype == torch.bool
         else torch.randint(0, 200, (B * K,) + shape, generator=g, device="cuda").to(dtype) for _ in range(3)]
    for turn in range(3):
        parents = torch.randint(0, K, (B, K), generator=g, device="cuda", dtype=torch.int32)
        if turn == 1:                          # a cycle through all
            parents = ((torch.arange(K, device="cuda") + 1) % K).int().repeat(B, 1)
        if turn == 2:
            parents[0, 0], parents[-1, -1] = -1, K  # no such beam: the row stays
        own = torch.arange(K, device="cuda").repeat(B, 1)
        p = torch.where((parents < 0) | (parents >= K), own, parents.long())
        rows = (p + torch.arange(0, B * K, K, device="cuda")[:, None]).reshape(-1)
        want = [t[rows] for t in x]
        beam_reorder(x, parents.contiguous())
        assert all(torch.equal(t, w) for t, w in zip(x, want))


def test_reorder_part_of_a_cache():
    """Positions 5 to 11 of a cache [sequences, heads, positions, size], and one kept [heads, sequences, ...]; the rest stays."""
    x = torch.randn(12, 4, 32, 48, device="cuda").bfloat16()
    y = torch.randn(4, 12, 9, device="cuda")
    parents = torch.tensor([[1, 2, 0, 0], [3, 2, 1, 0], [1, 1, 1, 1]], dtype=torch.int32, device="cuda")
    rows = (parents.long() + torch.arange(0, 12, 4, device="cuda")[:, None]).reshape(-1)
    want, wanty = x.clone(), y[:, rows]
    want[:, :, 5:12] = x[rows][:, :, 5:12]
    beam_reorder([x[:, :, 5:12], y.transpose(0, 1)], parents)
    assert torch.equal(x, want) and torch.equal(y, wanty)
    beam_reorder([torch.zeros(0, 4, device="cuda")], parents[:0].contiguous())
    with pytest.raises(ValueError, match="same memory"):
        beam_reorder([x, y.transpose(0, 1), x], parents)
    many = [torch.full((12, 3), float(i), device="cuda") for i in range(100)]
    many[99] = torch.arange(36.0, device="cuda").reshape(12, 3)
    want = many[99][rows]
    beam_reorder(many, parents)
    assert torch.equal(many[99], want)
