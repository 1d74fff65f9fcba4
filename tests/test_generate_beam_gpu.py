"""GPU suite: beam search of Llama handles against a search over the oracle's logits, every beam read anew from its first token."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT
from llama3_np_b200 import Llama, ModelArgs, _cabi
from llama3_np_b200.synth import make_weights
from oracle import ref_llama3 as orc

pytestmark = pytest.mark.gpu
F32_TOL, BF16_TOL = 1e-4, 3e-2          # of the logits, relative to the largest (test_parity_gpu.py)


def _args(heads, kv, dim, layers=2, vocab=300, seq=48, batch=8, **kw):
    return ModelArgs(dim=dim, n_layers=layers, n_heads=heads, n_kv_heads=kv, vocab_size=vocab, max_seq_len=seq, max_batch_size=batch, **kw)


def _log_probs(w, args, seqs):
    """log softmax of the next token for sequences of one length, in float64."""
    o = orc.OracleLlama(w, ModelArgs(**{**args.__dict__, "max_batch_size": len(seqs), "dtype": "float32"}))
    x = o(np.asarray(seqs), 0)[:, -1]
    return x - x.max(-1, keepdims=True) - np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)), np.abs(x).max()


def _search(w, args, prompt, beams, new, eos=None):
    """[(score, tokens)] by the definition; ended beams keep their score and only repeat eos.  And the largest |logit| seen.
    None where the logits' tolerance leaves open which beams live on."""
    live, top = [(0.0, [], False)], 0.0
    for _ in range(new):
        lp, big = _log_probs(w, args, [list(prompt) + t for _, t, _ in live])
        top = max(top, big)
        cand = []
        for k, (s, t, d) in enumerate(live):
            if d:
                cand.append((-s, k, eos))
            else:
                cand += [(-(s + lp[k, v]), k, int(v)) for v in np.argsort(-lp[k], kind="stable")[:beams + 1]]
        cand.sort()
        # which beams live on must not hang on the logits' tolerance (their order among one another may: it changes nothing that follows)
        if len(cand) > beams and cand[beams][0] - cand[beams - 1][0] <= 2 * 2 * (len(live[0][1]) + 1) * F32_TOL * top:
            return None
        live = [(-c[0], live[c[1]][1] + [c[2]], live[c[1]][2] or c[2] == eos) for c in cand[:beams]]
    return [(s, t) for s, t, _ in live], top


def _decided(w, args, vocab, count, length, beams, new, seed, eos=None):
    """`count` prompts whose search the logits' tolerance leaves no choice, with what it finds."""
    rng, prompts, found = np.random.default_rng(seed), [], []
    while len(prompts) < count:
        p = rng.integers(3, vocab, length)
        f = _search(w, args, p, beams, new, eos)
        if f is not None:
            prompts.append(p)
            found.append(f)
    return np.array(prompts), found


def _same(tokens, scores, want, new, top, eos=None, lengths=None):
    """The oracle's beams, each with its score (a log probability is off by at most twice a logit), best first."""
    score = {tuple(_cut(t, eos)): s for s, t in want}
    for j, (t, s) in enumerate(zip(tokens.tolist(), scores)):
        n = len(t) if lengths is None else int(lengths[j])
        assert tuple(t[:n]) in score and all(x == eos for x in t[n:]), (t, sorted(score))
        assert abs(s - score.pop(tuple(t[:n]))) <= new * 2 * F32_TOL * top
    assert not score and (np.diff(scores) <= 0).all()


def _cut(tokens, eos):
    return tokens[:tokens.index(eos) + 1] if eos in tokens else tokens


@pytest.mark.parametrize("heads,kv,dim,B,K", [(4, 4, 64, 2, 3), (8, 2, 256, 1, 4), (6, 3, 288, 3, 2), (4, 1, 512, 2, 4), (6, 6, 288, 2, 8)])
def test_equals_search_over_the_oracle(heads, kv, dim, B, K):
    args = _args(heads, kv, dim, vocab=61, batch=B * K)
    w = make_weights(args, 2 * dim, seed=dim + K)
    prompts, found = _decided(w, args, 61, B, 7, K, 5, K)
    m = Llama(w, args)
    tokens, scores, lengths = m.generate_beam(prompts, K, 5)
    again = m.generate_beam(prompts, K, 5)
    m.close()
    assert np.array_equal(tokens, again[0]) and np.array_equal(scores, again[1])
    for b in range(B):
        want, top = found[b]
        _same(tokens[b], scores[b], want, 5, top)
    assert (lengths == 5).all()


def test_one_beam_is_greedy_and_the_cache_survives():
    """One beam is the greedy run at contiguous positions, over a captured step; greedy runs on a fresh cache before and after agree."""
    args = _args(6, 6, 288, layers=3, vocab=500, seq=64, batch=4)
    w = make_weights(args, 768, seed=5)
    ids = np.random.default_rng(5).integers(3, 500, (4, 9))
    m = Llama(w, args)
    before = m.generate_all(ids, 40)
    want = np.stack(m.generate_ragged(list(ids), 30, schedule="simple"))
    tokens, _, _ = m.generate_beam(ids, 1, 30)
    assert np.array_equal(tokens[:, 0], want)
    assert m.generate_beam(ids[:2], 2, 30)[0].shape == (2, 2, 30)
    m.reset_cache()          # the reference's schedule skips slot L, so its run sees what was there before
    assert np.array_equal(m.generate_all(ids, 40), before)
    assert np.array_equal(m.generate_beam(ids, 1, 30)[0], tokens)
    m.close()


@pytest.mark.parametrize("K", [1, 3])
def test_end_token(K):
    args = _args(4, 2, 64, vocab=23, batch=2 * K)
    w = make_weights(args, 160, seed=9)
    first, found = _decided(w, args, 23, 1, 4, K, 6, 2)
    eos = found[0][0][0][1][2]                    # its best beam ends at its third token at the latest
    prompts, found = _decided(w, args, 23, 2, 4, K, 6, 2, eos)
    m = Llama(w, args)
    tokens, scores, lengths = m.generate_beam(prompts, K, 6, eos_id=eos)
    long = m.generate_beam(prompts, K, 20, eos_id=eos)
    m.close()
    for b in range(2):
        want, top = found[b]
        _same(tokens[b], scores[b], want, 6, top, eos, lengths[b])
    assert long[0].shape == (2, K, 20) and (long[2] <= 20).all()


def test_length_penalty_sorts():
    args = _args(4, 2, 64, vocab=23, batch=4)
    w = make_weights(args, 160, seed=9)
    prompt = np.random.default_rng(2).integers(3, 23, (1, 4))
    m = Llama(w, args)
    free, _, _ = m.generate_beam(prompt, 4, 6)
    eos = int(free[0, 0, 2])
    t0, s0, n0 = m.generate_beam(prompt, 4, 6, eos_id=eos)
    t1, s1, n1 = m.generate_beam(prompt, 4, 6, eos_id=eos, length_penalty=1.0)
    _, s2, n2 = m.generate_beam(prompt, 4, 6, eos_id=eos, length_penalty=1e30)   # 1^x = 1, any other length's power is infinite
    m.close()
    raw = {tuple(t[:n]): s for t, s, n in zip(t0[0].tolist(), s0[0], n0[0])}
    assert (np.diff(s0[0]) <= 0).all() and (np.diff(s1[0]) <= 0).all()
    for t, s, n in zip(t1[0].tolist(), s1[0], n1[0]):
        assert abs(s - raw[tuple(t[:n])] / n) <= 1e-6 * abs(s)
    assert ((s2[0] == 0) == (n2[0] > 1)).all() and (np.diff(s2[0]) <= 0).all()


@pytest.mark.parametrize("heads,kv,dim,K", [(8, 2, 512, 4), (4, 4, 256, 10), (2, 1, 256, 3)])
def test_bf16_scores_are_those_of_the_tokens(heads, kv, dim, K):
    """bf16 mode: the score of every beam is the sum of its tokens' log probabilities, and the best beam's is no worse than greedy's."""
    args = _args(heads, kv, dim, vocab=257, batch=2 * K, dtype="bfloat16")
    w = make_weights(args, 2 * dim, seed=dim)
    ids = np.random.default_rng(1).integers(3, 257, (2, 11))
    m = Llama(w, args)
    tokens, scores, _ = m.generate_beam(ids, K, 6)
    greedy, gs, _ = m.generate_beam(ids, 1, 6)
    m.close()
    for b in range(2):
        total, top = np.zeros(K), 0.0
        for s in range(6):
            lp, big = _log_probs(w, args, [list(ids[b]) + tokens[b, k, :s].tolist() for k in range(K)])
            total += lp[np.arange(K), tokens[b, :, s]]
            top = max(top, big)
        # a log probability is off by at most twice the largest error of a logit
        np.testing.assert_allclose(scores[b], total, rtol=0, atol=6 * 2 * BF16_TOL * top)
        assert len({tuple(t) for t in tokens[b].tolist()}) == K
        assert scores[b, 0] >= gs[b, 0] - 6 * 2 * BF16_TOL * top


def test_odd_lengths_and_limits():
    """max_seq_len that is no multiple of 4, a prompt of one token, the last position, as many beams as tokens."""
    args = _args(4, 2, 64, vocab=5, seq=13, batch=10)
    w = make_weights(args, 160, seed=3)
    m = Llama(w, args)
    tokens, scores, _ = m.generate_beam([[2], [4]], 5, 13)
    found = _search(w, args, [2], 5, 2)
    assert found is not None
    want, top = found
    got, gs, _ = m.generate_beam([[2], [4]], 5, 2)
    _same(got[0], gs[0], want, 2, top)
    assert tokens.shape == (2, 5, 13) and np.isfinite(scores).all() and (tokens < 5).all() and (tokens >= 0).all()
    one, _, _ = m.generate_beam([[2] * 13], 3, 1)
    lp, _ = _log_probs(w, args, [[2] * 13])
    assert one[0, :, 0].tolist() == np.argsort(-lp[0], kind="stable")[:3].tolist()
    m.close()


def test_refusals():
    args = _args(4, 2, 64, vocab=30, seq=16, batch=6)
    m = Llama(make_weights(args, 160, seed=1), args)
    ids = np.array([[1, 2, 3], [4, 5, 6]])
    for a, kw in [((ids, 4, 4), {}), ((ids, 0, 4), {}), ((ids, -1, 4), {}), ((ids, 3, 15), {}), ((ids, 3, 0), {}), ((ids, 3, -2), {}),
                  ((ids, 3, 4), dict(eos_id=30)), ((ids, 3, 4), dict(eos_id=-1)), ((ids, 3, 4), dict(length_penalty=-0.5)),
                  ((ids, 3, 4), dict(length_penalty=float("nan"))), ((ids, 3, 4), dict(length_penalty=float("inf"))), (([[1, 30]], 3, 4), {}), ((ids[0], 3, 4), {})]:
        with pytest.raises(ValueError):
            m.generate_beam(*a, **kw)
    assert m.generate_beam(ids, 3, 14)[0].shape == (2, 3, 14)
    m.close()


def test_layer_lists_are_refused():
    from test_risalix_gpu import attn, build, config
    m, _ = build(config([attn()]), max_seq_len=16, max_batch_size=2)
    ids, tokens = np.array([[1, 2, 3]], np.int32), np.zeros((1, 2, 2), np.int64)
    scores, lengths = np.zeros((1, 2), np.float32), np.zeros((1, 2), np.int32)
    rc = _cabi.lib().l3_generate_beam(m._h, _cabi.i32p(ids), 1, 3, 2, 2, -1, 0.0, _cabi.i64p(tokens), _cabi.f32p(scores), _cabi.i32p(lengths))
    assert rc == _cabi.L3_EINVAL and b"layer-list" in _cabi.lib().l3_last_error(m._h)
    m.close()


def test_command_line(tmp_path):
    args = _args(4, 2, 64, vocab=61, batch=6)
    w = make_weights(args, 160, seed=11)
    np.savez(tmp_path / "model.npz", **w)
    fields = {k: getattr(args, k) for k in ("dim", "n_layers", "n_heads", "n_kv_heads", "vocab_size")}
    (tmp_path / "config.json").write_text(json.dumps({"architecture": "Llama", "args": fields}))
    (tmp_path / "prompts.txt").write_text("5 17 3\n9 8 7\n")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "generate"), "--model", str(tmp_path), "--dtype", "float32",
                        "--batch-file", str(tmp_path / "prompts.txt"), "--new", "6", "--beams", "3"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    m = Llama(w, args)
    want, _, _ = m.generate_beam([[5, 17, 3], [9, 8, 7]], 3, 6)
    m.close()
    assert [list(map(int, line.split())) for line in r.stdout.strip().splitlines()[-2:]] == want[:, 0].tolist()
