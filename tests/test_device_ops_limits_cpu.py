"""CPU suite: numbers and arguments at the edge of what the operators on device buffers and beam search take."""
import numpy as np
import pytest
import torch

from llama3_np_b200 import Llama, ModelArgs, beam_reorder, copy_pages


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
