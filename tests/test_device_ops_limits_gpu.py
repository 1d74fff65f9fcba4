"""GPU suite: the operators on device buffers and beam search at the edge of what they take."""
import numpy as np
import pytest
import torch

from llama3_np_b200 import Llama, ModelArgs, _cabi, beam_reorder, copy_pages
from llama3_np_b200.synth import make_weights

pytestmark = pytest.mark.gpu


def test_beam_search_refuses_more_tokens_than_the_cache_holds():
    """Also where the sum with the prompt's length passes 32 bits: refused on the host, before anything is enqueued."""
    args = ModelArgs(dim=64, n_layers=1, n_heads=2, n_kv_heads=1, vocab_size=30, max_seq_len=16, max_batch_size=6)
    m = Llama(make_weights(args, 160, seed=1), args)
    lib, before = _cabi.lib(), m.launch_count()
    scores, lengths = np.zeros((1, 2), np.float32), np.zeros((1, 2), np.int32)
    tokens = np.full((1, 2, 16), -7, np.int64)
    for L in (1, 2, 9, 16):
        ids = np.ones((1, L), np.int32)
        for new in (2 ** 31 - 1, 2 ** 31 - 16, 18 - L):
            rc = lib.l3_generate_beam(m._h, _cabi.i32p(ids), 1, L, 2, new, 3, 0.0, _cabi.i64p(tokens), _cabi.f32p(scores), _cabi.i32p(lengths))
            assert rc == _cabi.L3_EINVAL and b"max_seq_len" in lib.l3_last_error(m._h)
        assert m.launch_count() == before and (tokens == -7).all()
    assert m.generate_beam(np.ones((1, 9), np.int64), 2, 8)[0].shape == (1, 2, 8)
    m.close()


def test_positions_near_2_31_are_refused():
    """A position or a number of tokens whose sum with the prompt's length passes 32 bits, by the calls of a handle that take one."""
    args = ModelArgs(dim=64, n_layers=1, n_heads=2, n_kv_heads=1, vocab_size=30, max_seq_len=16, max_batch_size=2)
    m = Llama(make_weights(args, 160, seed=1), args)
    lib, before = _cabi.lib(), m.launch_count()
    logits, out, lens = np.zeros((1, 30), np.float32), np.full((1, 16), -7, np.int64), np.array([9], np.int32)
    ids = np.ones((1, 9), np.int32)
    for start in (2 ** 31 - 1, 2 ** 31 - 9, 8):
        assert lib.l3_forward(m._h, _cabi.i32p(ids), 1, 9, start, _cabi.f32p(logits), None) == _cabi.L3_EINVAL
    for new in (2 ** 31 - 1, 2 ** 31 - 8, 8):
        assert lib.l3_generate_ragged(m._h, _cabi.i32p(ids), _cabi.i32p(lens), 1, 9, new, 0, -1, _cabi.i64p(out)) == _cabi.L3_EINVAL
    assert m.launch_count() == before and (out == -7).all()
    assert lib.l3_forward(m._h, _cabi.i32p(ids), 1, 9, 7, _cabi.f32p(logits), None) == _cabi.L3_OK
    assert lib.l3_generate_ragged(m._h, _cabi.i32p(ids), _cabi.i32p(lens), 1, 9, 7, 0, -1, _cabi.i64p(out)) == _cabi.L3_OK
    m.close()


@pytest.mark.parametrize("as_what", [lambda x: (t for t in x), lambda x: dict(enumerate(x)).values(), iter, tuple])
def test_states_from_any_iterable(as_what):
    """Tensors that come from a generator or a dict's values are reordered and copied once, and count as modified."""
    x = [torch.randn(6, 5, device="cuda"), torch.arange(6, device="cuda")]
    parents = torch.tensor([[2, 0, 0], [1, 2, 2]], dtype=torch.int32, device="cuda")
    rows = (parents.long() + torch.tensor([[0], [3]], device="cuda")).reshape(-1)
    want, version = [t[rows] for t in x], [t._version for t in x]
    beam_reorder(as_what(x), parents)
    assert all(torch.equal(t, w) for t, w in zip(x, want)) and all(t._version > v for t, v in zip(x, version))
    src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (1, 4))
    copy_pages(as_what(x), src, dst)
    assert all(torch.equal(t[4], w[1]) for t, w in zip(x, want))


@pytest.mark.parametrize("width", [3, 4096, 50000])
def test_tensors_of_different_alignment(width):
    """Bytes, 2-, 4-, 8- and 16-byte pieces in one call, few of them (one launch) and many (one for each size); a hundred tensors."""
    B, K = 4, 5
    g = torch.Generator(device="cuda").manual_seed(width)
    ints = lambda shape, dtype: torch.randint(-100, 100, shape, generator=g, device="cuda").to(dtype)
    x = [ints((B * K, width, 8), torch.float32), ints((B * K,), torch.bool), ints((B * K, width), torch.int8), ints((B * K, 2 * width + 1), torch.int16),
         ints((B * K, 5), torch.int32), ints((B * K, 3), torch.int64), torch.zeros(B * K, 0, device="cuda")]
    x += [ints((B * K, 1 + i % 7), (torch.int8, torch.int32, torch.float64)[i % 3]) for i in range(93)]
    parents = torch.randint(0, K, (B, K), generator=g, device="cuda").int()
    rows = (parents.long() + torch.arange(0, B * K, K, device="cuda")[:, None]).reshape(-1)
    want = [t[rows] for t in x]
    beam_reorder(x, parents)
    assert all(torch.equal(t, w) for t, w in zip(x, want))
    src, dst = torch.tensor([3, 0, -1], device="cuda").int(), torch.tensor([7, 19, 2], device="cuda").int()
    copy_pages(x, src, dst)
    for w in want:
        w[7], w[19] = w[3].clone(), w[0].clone()
    assert all(torch.equal(t, w) for t, w in zip(x, want))


def test_a_refused_tensor_leaves_the_others_as_they_were():
    lib = _cabi.lib()
    x = torch.arange(70 * 6, device="cuda").reshape(70, 6).contiguous()
    parents = torch.tensor([[1, 2, 0], [2, 1, 0]], dtype=torch.int32, device="cuda")
    rows = (_cabi.L3Rows * 71)(*(_cabi.L3Rows(x[i].data_ptr(), 6, 8, 1, 0, 8) for i in range(70)), _cabi.L3Rows(x.data_ptr() + 1, 6, 1 << 31, 1, 0, 1 << 31))
    assert lib.l3_beam_reorder(0, None, rows, 71, parents.data_ptr(), 2, 3) == _cabi.L3_EINVAL
    torch.cuda.synchronize()
    assert torch.equal(x, torch.arange(70 * 6, device="cuda").reshape(70, 6))
