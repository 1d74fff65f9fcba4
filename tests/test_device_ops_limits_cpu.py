"""CPU suite: numbers and arguments at the edge of what the operators on device buffers and beam search take."""
import numpy as np
import pytest

from llama3_np_b200 import Llama, ModelArgs


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
