"""CPU suite: numbers and arguments at the edge of what the operators on device buffers and beam search take."""
import ctypes as C

import numpy as np
import pytest
import torch

from llama3_np_b200 import Llama, ModelArgs, _cabi, beam_reorder, beam_select, copy_pages, paged_attention, paged_write


class _Library:
    """Stands in for the library: a call that reaches it is recorded, and fails."""

    def __init__(self):
        self.calls = []

    def l3_generate_beam(self, *args):
        self.calls.append(args)
        raise AssertionError("the call was to be refused")

    def l3_destroy(self, handle):
        return 0


def _model():
    m = Llama.__new__(Llama)
    m.args, m._lib, m._h = ModelArgs(dim=64, n_layers=1, n_heads=1, vocab_size=30, max_seq_len=16, max_batch_size=6), _Library(), None
    return m


@pytest.mark.parametrize("beams,new,kw", [
    (2 ** 32 + 2, 4, {}), (-2 ** 32 + 2, 4, {}), (7, 4, {}), (0, 4, {}), (2, 2 ** 32 + 4, {}), (2, 2 ** 31 - 1, {}), (2, 17, {}), (2, 0, {}),
    (2, 4, dict(eos_id=2 ** 32 + 2)), (2, 4, dict(eos_id=30)), (2, 4, dict(eos_id=-1)), (2, 4, dict(eos_id=-2 ** 32 + 2))])
def test_beam_search_refuses_what_a_call_would_cut_to_32_bits(beams, new, kw):
    m = _model()
    with pytest.raises(ValueError, match="eos_id" if kw else "beams" if new == 4 else "max_new_tokens"):
        m.generate_beam(np.array([[1, 2, 3]]), beams, new, **kw)
    assert not m._lib.calls


ITERABLES = [list, tuple, iter, lambda x: (t for t in x), lambda x: map(lambda t: t, x), lambda x: dict(enumerate(x)).values(), lambda x: x[0]]


@pytest.mark.parametrize("as_what", ITERABLES)
def test_any_iterable_of_tensors_is_checked(as_what):
    """A generator's tensors, which can be seen once only, are refused as a list's are: no address of the host reaches a kernel."""
    idx, parents = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    states = lambda: [torch.zeros(6, 4), torch.zeros(6, 7)]
    with pytest.raises(ValueError, match="pools must be on a CUDA device"):
        copy_pages(as_what(states()), idx, idx)
    with pytest.raises(ValueError, match="states must be on a CUDA device"):
        beam_reorder(as_what(states()), parents)


def test_what_no_tensors_come_from_is_refused():
    idx, parents = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    for states, error in [((x for x in ()), ValueError), ({}.values(), ValueError), (7, TypeError), (None, TypeError), ([7], ValueError), ("ab", ValueError)]:
        with pytest.raises(error):
            copy_pages(states, idx, idx)
    for states, error in [((x for x in ()), ValueError), (7, TypeError), (["a"], ValueError)]:
        with pytest.raises(error):
            beam_reorder(states, parents)


def _rows(*tensors):
    return (_cabi.L3Rows * len(tensors))(*(_cabi.L3Rows(*t) for t in tensors))


def test_every_tensor_is_checked_ahead_of_the_first_launch():
    """A tensor that is refused behind more of them than one launch takes: nothing was enqueued, so there is no device to ask for."""
    lib, some = _cabi.lib(), C.c_void_p(0x1000)
    fine = [(0x100000 + 64 * i, 6, 64, 1, 0, 64) for i in range(70)]
    for bad, text in [((0x1, 6, 1 << 31, 1, 0, 1 << 31), b"too long"), ((0x10, 6, 1 << 40, 1 << 30, 64, 64), b"too long"), ((0, 6, 64, 1, 0, 64), b"no data"),
                      ((0x10, 5, 64, 1, 0, 64), b"5 rows"), ((0x10, 6, 64, -1, 0, 64), b"bad sizes")]:
        rows = _rows(*fine, bad)
        assert lib.l3_beam_reorder(0, None, rows, 71, some, 2, 3) == _cabi.L3_EINVAL and text in lib.l3_last_error(None)
        assert lib.l3_copy_rows(0, None, rows, 71, some, some, 2) == _cabi.L3_EINVAL and text in lib.l3_last_error(None)


def test_a_long_row_beside_odd_bytes():
    """What a row may hold hangs on its own alignment alone."""
    rows = _rows((0x1000, 6, 1 << 33, 1, 0, 1 << 33), (0x3, 6, 13, 1, 0, 13))
    assert _cabi.lib().l3_copy_rows(0, None, rows, 2, None, None, 0) == _cabi.L3_OK


def test_forward_mode_gradients_are_refused():
    """A tangent that a call would drop is as wrong as a gradient without its backward pass."""
    from torch.autograd import forward_ad
    pool, table, idx = torch.zeros(5, 2, 16, 64), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with forward_ad.dual_level():
        dual = lambda *shape: forward_ad.make_dual(torch.zeros(*shape), torch.ones(*shape))
        calls = [lambda: paged_attention(dual(2, 8, 64), pool, pool, table, idx),
                 lambda: paged_attention(torch.zeros(2, 8, 64), pool, dual(5, 2, 16, 64), table, idx),
                 lambda: paged_attention(dual(2, 8, 128)[..., :64], pool, pool, table, idx),
                 lambda: paged_write(dual(2, 4, 2, 64), torch.zeros(2, 4, 2, 64), pool, pool, table, idx),
                 lambda: copy_pages([pool, dual(5, 3)], idx, idx), lambda: beam_reorder(dual(4, 3), table),
                 lambda: beam_select(dual(2, 3, 50), torch.zeros(2, 3))]
        for call in calls:
            for grad in (True, False):  # no_grad() is of the other mode
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    call()
            with forward_ad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA device"):
                call()
        with pytest.raises(ValueError, match="CUDA device"):
            beam_select(forward_ad.unpack_dual(dual(2, 3, 50)).primal, torch.zeros(2, 3))
