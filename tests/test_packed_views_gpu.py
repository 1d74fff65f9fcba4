"""GPU suite: the rows of a cache's view, asked for on one stream and used on another, or in a capture."""
import pytest
import torch

from llama3_np_b200 import PagedCache
from llama3_np_b200.packed import PackedStep

pytestmark = pytest.mark.gpu


def _cache():
    cache = PagedCache(layers=1, kv_heads=2, head_dim=64, pages=40)
    a, b = cache.open(), cache.open()
    cache.extend([a, b], [20, 3])
    return cache, [a, b]


def test_rows_made_on_one_stream_are_there_on_every_other():
    cache, seqs = _cache()
    view = cache.extend(seqs, [30, 1])
    want = [view.starts.clone(), view.positions.clone(), view.slots.clone()]
    late = cache.view(seqs, [20, 3])
    made = late._packed

    def slowly():
        """The same, long after the call has returned."""
        step = made()
        out = PackedStep(*(torch.full_like(t, -9) for t in step))
        torch.cuda._sleep(200_000_000)
        for to, t in zip(out, step):
            to.copy_(t)
        return out

    late._packed = slowly
    with torch.cuda.stream(torch.cuda.Stream()):
        late.starts
    with torch.cuda.stream(torch.cuda.Stream()):
        got = [late.starts.clone(), late.positions.clone(), late.slots.clone()]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_rows_first_asked_for_in_a_capture_are_refused_and_the_capture_goes_on():
    cache, seqs = _cache()
    view = cache.extend(seqs, [30, 1])
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="ahead of the capture"):
            view.positions
        x += 1
    graph.replay()
    torch.cuda.synchronize()
    assert bool((x == 1).all())
    q, k, v = (torch.randn(31, n, 64, device="cuda").bfloat16() for n in (4, 2, 2))
    cache.write_packed(0, view, q, k, v, torch.zeros(32, dtype=torch.float64, device="cuda"))   # and asked for ahead of one they are good in it
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend_packed(0, view, q, out=out)
    graph.replay()
    assert torch.equal(out, cache.attend_packed(0, view, q, out=torch.zeros_like(q)))
