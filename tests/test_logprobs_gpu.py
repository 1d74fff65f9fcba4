"""GPU suite: log probabilities of given tokens, entropy and the most likely tokens, against their formulas in 64 bits."""
import math

import pytest
import torch

from llama3_np_b200 import token_logprobs

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def formula(x, tokens, top):
    x = x.double()
    none = (x == -math.inf).all(-1)
    p = torch.log_softmax(x, -1)
    p = torch.where(none[:, None], torch.full_like(p, -math.inf), p)
    entropy = -torch.where(p > -math.inf, p.exp() * p, torch.zeros_like(p)).sum(-1)
    entropy = torch.where(p.isnan().any(-1), torch.full_like(entropy, math.nan), entropy)
    V = x.shape[1]
    lp = p.gather(1, tokens.long().clamp(0, V - 1)[:, None])[:, 0]
    lp = torch.where(tokens < 0, torch.zeros_like(lp), torch.where(tokens >= V, torch.full_like(lp, math.nan), lp))
    val, idx = x.nan_to_num(-math.inf, posinf=math.inf, neginf=-math.inf).sort(dim=1, descending=True, stable=True)
    val, idx = val[:, :top], idx[:, :top]
    best = torch.where(val > -math.inf, p.gather(1, idx), torch.full_like(val, -math.inf))
    return lp, entropy, best, torch.where(val > -math.inf, idx, -1)


def same(got, want, tol):
    assert got.dtype == torch.float32
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and torch.equal(got[want.isinf()], want[want.isinf()])
    fine = want.isfinite()
    err = ((got - want).abs() / tol.expand_as(want) if tol.dim() == want.dim() else (got - want).abs() / tol[:, None])[fine]
    assert err.numel() == 0 or float(err.max()) <= 1, f"{float(err.max()):.3f} of the bound"


def check(x, tokens, top=0):
    got = token_logprobs(x, tokens, top=top, entropy=True)
    lp, entropy, best, idx = formula(x, tokens, top)
    finite = torch.where(x.isfinite(), x.double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    spread = finite.amax(-1) - finite.amin(-1)
    # a logit's distance to the largest is rounded once, and once as a multiple of log 2 (2^-23 of it together); exponentials 2^-21; every thread
    # adds up at most V / 64 of them, then five and five sums; the logarithm, two differences of up to the spread
    V = x.shape[1]
    sums = (V / 64 + 30) * 2.0 ** -24 + 2.0 ** -21
    tol = spread * 2.0 ** -22 + sums + 2.0 ** -20
    same(got.logprobs, lp, tol)
    # an entropy's terms are p d: as many roundings of each, and the moves of the maximum
    most = torch.where(entropy.isfinite(), entropy, torch.zeros_like(entropy))
    same(got.entropy, entropy, (spread + most + 1) * (2 * sums + 2.0 ** -20))
    if top:
        same(got.top_logprobs, best, tol)
        assert got.top_tokens.dtype == torch.int32 and torch.equal(got.top_tokens.long(), idx)
        plain = token_logprobs(x, tokens, top=top)
        assert plain.entropy is None and torch.equal(plain.top_tokens, got.top_tokens) and torch.equal(plain.logprobs.isnan(), got.logprobs.isnan())
    else:
        assert got.top_logprobs is None and got.top_tokens is None
    return got


def logits(seed, rows, vocab, kind, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * scale).to(TYPES[kind])
    return x, torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (2, 500), (70, 1000), (1, 32000), (7, 50257), (40, 128256), (300, 32001), (1000, 77), (70000, 9)])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_sizes(kind, rows, vocab, top):
    x, t = logits(rows + vocab, rows, vocab, kind)
    check(x, t, min(top, vocab))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("top", [0, 20])
@pytest.mark.parametrize("scale", [0.0, 0.01, 30.0])
def test_flat_and_peaked(kind, top, scale):
    """Equal logits alone (every one passes any bound), nearly equal ones, one token that has all."""
    x, t = logits(5, 9, 40000, kind, scale)
    check(x, t, top)


@pytest.mark.parametrize("kind", list(TYPES))
def test_rows_of_any_stride_and_start(kind):
    whole, t = logits(6, 12, 9000, kind)
    for at in range(9):
        check(whole[:, at:at + 8003], t.clamp(max=8002), 7)
        check(whole[::3, at:at + 13], t[::3].contiguous().clamp(max=12), 3)
    check(whole[:1].expand(12, 9000), t, 4)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [40, 30000])
def test_tokens_that_are_banned_and_numbers_that_are_none(kind, vocab):
    x, t = logits(7, 14, vocab, kind)
    lowest = torch.finfo(TYPES[kind]).min
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 17] = 3.0
    x[2, ::2] = -math.inf
    x[3, 5] = math.nan
    x[4, 6] = math.inf
    x[5, 1:] = lowest                                       # a mask of the type's lowest value
    x[6] = lowest
    x[7, :-3] = -math.inf
    x[8] = math.nan
    x[9, 0], x[9, 1] = 0.0, -0.0
    t[0], t[1], t[2], t[7], t[10], t[11], t[12], t[13] = 3, 17, 4, 0, -1, vocab, 2 ** 31 - 1, -2 ** 31
    check(x, t, 8)
    check(x, t, 0)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("top", [20, 64])
def test_equal_logits_come_by_token(kind, top):
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randint(0, 12, (33, 60001), generator=g, device="cuda").to(TYPES[kind])    # thousands of each
    check(x, torch.zeros(33, dtype=torch.int32, device="cuda"), top)
    few = torch.full((4, 60001), -3.0, device="cuda").to(TYPES[kind])
    few[:, ::6007] = 1.0                                                              # ten of them
    check(few, torch.zeros(4, dtype=torch.int32, device="cuda"), top)
    rising = torch.arange(60001, device="cuda").div(8000).expand(3, 60001).contiguous()
    check(rising.to(TYPES[kind]), torch.zeros(3, dtype=torch.int32, device="cuda"), top)


def test_no_rows():
    got = token_logprobs(torch.zeros(0, 50, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), top=3, entropy=True)
    assert got.logprobs.shape == (0,) and got.entropy.shape == (0,) and got.top_logprobs.shape == (0, 3) and got.top_tokens.shape == (0, 3)


def test_rows_beyond_32_bits():
    """The last row begins 2^31 logits on."""
    x = torch.zeros(70, 1 << 25, dtype=torch.bfloat16, device="cuda")[:, :8000]
    x[69] = torch.randn(8000, device="cuda").bfloat16()
    check(x, torch.full((70,), 5, dtype=torch.int32, device="cuda"), 4)


def test_captured_and_on_another_stream():
    x, t = logits(9, 50, 32000, "f32")
    token_logprobs(x, t, top=5, entropy=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_logprobs(x, t, top=5, entropy=True)
    x.copy_(logits(10, 50, 32000, "f32")[0])
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = token_logprobs(x, t, top=5, entropy=True)
    torch.cuda.synchronize()
    want = check(x, t, 5)
    for a, b, c in zip(got, other, want):
        assert torch.equal(a, c) and torch.equal(b, c)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [100, 515, 3277, 4100, 9000])
@pytest.mark.parametrize("top", [33, 64])
@pytest.mark.parametrize("banned", [0.0, 0.97])
def test_rows_with_too_few_logits_for_a_warps_bound(kind, vocab, top, banned):
    x, t = logits(8, 5, vocab, kind)
    g = torch.Generator(device="cuda").manual_seed(9)
    check(x.masked_fill(torch.rand(x.shape, generator=g, device="cuda") < banned, -math.inf), t, top)
