"""GPU suite: log probabilities and entropy of rows in which one token has nearly all, by what fp32 can tell there."""
import math

import pytest
import torch

from llama3_np_b200 import token_logprobs

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("gap", [2.5, 4.0, 7.75, 7.9, 12.0, 30.0])
@pytest.mark.parametrize("vocab", [9000, 128256])
@pytest.mark.parametrize("rows", [2, 200])
@pytest.mark.parametrize("top", [0, 5])
def test_one_large_logit(kind, gap, vocab, rows, top):
    """Eight logits at a row's start and one that is `gap` larger behind them, at places of the same thread's and of others; no other token is allowed.

    The large one is what the sums end up against: it adds exactly 1, the others delta.  Sums of 1 to 2 are rounded by 2^-24 at most, and there is one for each
    thread that holds some of the eight: 16 bytes are a thread's, so fp32's eight are two threads' (1 + delta_1, and the whole of it + delta_2), 16-bit ones
    one's.  All else - exponentials 2^-22, arguments, sums, the logarithm, products, 2^-20 together - is relative to what the other tokens add."""
    step = 2.0 ** -23 if kind == "f32" else 2.0 ** -24
    x = torch.full((rows, vocab), -math.inf, device="cuda")
    base = torch.arange(rows, device="cuda") % 7 - 3.0
    for place in (2048, 4096, 8192):
        x[:, 8:] = -math.inf
        x[:, :8], x[:, place] = base[:, None], base + gap
        y, tokens = x.to(TYPES[kind]), torch.full((rows,), place, dtype=torch.int32, device="cuda")
        got = token_logprobs(y, tokens, top=top, entropy=True)
        p = torch.log_softmax(y.double(), -1)
        lp, entropy = p[:, place], -torch.where(p > -math.inf, p.exp() * p, 0.0).sum(-1)
        assert bool(((got.logprobs - lp).abs() <= step + lp.abs() * 2.0 ** -20).all())
        assert bool(((got.entropy - entropy).abs() <= step + entropy * 2.0 ** -20).all())
        if top:
            assert bool((got.top_tokens[:, 0] == place).all()) and torch.equal(got.top_logprobs[:, 0], got.logprobs)
