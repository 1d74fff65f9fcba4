"""CPU suite: what the operators on device buffers refuse, from Python and through the C-ABI, and the index arithmetic of rows."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

from conftest import ROOT
from llama3_np_b200 import _cabi, beam_reorder, beam_select, copy_pages, paged_attention, paged_write
from llama3_np_b200.paged import _ops


def _attn(**change):
    a = dict(q=torch.zeros(2, 8, 64, dtype=torch.bfloat16), k_pages=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16),
             v_pages=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16), page_table=torch.zeros(2, 2, dtype=torch.int32),
             lengths=torch.zeros(2, dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(2, 8, 64)[0]), "dimensions"),
    (dict(q=torch.zeros(2, 8, 64, dtype=torch.float16)), "cache's type or fp32"),
    (dict(q=torch.zeros(2, 7, 64, dtype=torch.bfloat16)), "heads over"),
    (dict(q=torch.zeros(2, 8, 128, dtype=torch.bfloat16)), "head size"),
    (dict(q=torch.zeros(2, 64, 8, dtype=torch.bfloat16).transpose(1, 2)), "contiguous"),
    (dict(k_pages=torch.zeros(5, 2, 12, 64, dtype=torch.bfloat16), v_pages=torch.zeros(5, 2, 12, 64, dtype=torch.bfloat16)), "power of two"),
    (dict(v_pages=torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)), "differ"),
    (dict(v_pages=torch.zeros(5, 2, 16, 64)), "type"),
    (dict(k_pages=torch.zeros(5, 2, 16, 65, dtype=torch.bfloat16)[..., 1:]), "16 bytes"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32)), "rows"),
    (dict(page_table=torch.zeros(2, 2, dtype=torch.int64)), "type"),
    (dict(page_table=torch.zeros(2, 2, dtype=torch.int32).T), "contiguous"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)[::2]), "contiguous"),
    (dict(k_new=torch.zeros(2, 2, 64, dtype=torch.bfloat16)), "go together"),
    (dict(k_new=torch.zeros(2, 2, 64), v_new=torch.zeros(2, 2, 64)), "type"),
    (dict(out=torch.zeros(2, 8, 64)), "out"),
    (dict(), "CUDA device"),
])
def test_attention_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        paged_attention(**_attn(**change))


def test_write_refuses():
    pool = torch.zeros(5, 2, 16, 64)
    k, table, start = torch.zeros(3, 4, 2, 64), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for args, text in [((k, k[:2], pool, pool, table, start), "must be"), ((k, k, pool, pool, table[:2], start), "rows"),
                       ((k, k, pool, pool, table, start[:2]), "start"), ((k, k, pool, pool, table, start, start[:1]), "count"),
                       ((k.half(), k.half(), pool, pool, table, start), "type"), ((k, k, pool, pool, table, start), "CUDA device")]:
        with pytest.raises(ValueError, match=text):
            paged_write(*args)
    odd = torch.zeros(5, 1, 16, 2)
    with pytest.raises(ValueError, match="16 bytes"):
        paged_write(torch.zeros(3, 4, 1, 2), torch.zeros(3, 4, 1, 2), odd, odd, table, start)


def test_rows_refuse():
    idx = torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(6, 2, 8, 4)
    for args, text in [(([], idx, idx), "no pools"), (([pool, pool[:5]], idx, idx), "pages"), (([pool], idx.long(), idx), "type"),
                       (([pool], idx, idx[:1]), "dst"), (([pool.expand(3, 6, 2, 8, 4)], idx, idx), "overlap"),
                       (([pool[:, :, ::2, ::2]], idx, idx), "equal"), (([pool], idx, idx), "CUDA device")]:
        with pytest.raises(ValueError, match=text):
            copy_pages(*args)
    par = torch.zeros(2, 3, dtype=torch.int32)
    for args, text in [(([pool[:5]], par), "rows for"), (([pool], par[0]), "dimensions"), (([pool], par.long()), "type"),
                       (([torch.zeros(257)], torch.zeros(1, 257, dtype=torch.int32)), "beams"), (([pool], par), "CUDA device")]:
        with pytest.raises(ValueError, match=text):
            beam_reorder(*args)


def test_select_refuses():
    x, s = torch.zeros(2, 3, 50), torch.zeros(2, 3)
    d = torch.zeros(2, 3, dtype=torch.bool)
    for args, kw, text in [((x[0], s), {}, "dimensions"), ((x.double(), s), {}, "type"), ((x, s[:1]), {}, "scores"),
                           ((x, s.double()), {}, "type"), ((x, s, 65), {}, "best"), ((x, s, 0), {}, "best"),
                           ((torch.zeros(1, 257, 4), torch.zeros(1, 257)), {}, "beams"), ((x, s), {"done": d}, "eos_id"),
                           ((x, s), {"done": d, "eos_id": 50}, "eos_id"), ((x, s), {"eos_id": -1}, "eos_id"),
                           ((x, s), {"done": d[:1], "eos_id": 1}, "done"), ((x.transpose(1, 2), torch.zeros(2, 50)), {}, "contiguous"),
                           ((x, s), {}, "CUDA device")]:
        with pytest.raises(ValueError, match=text):
            beam_select(*args, **kw)


def test_gradients_are_refused():
    """None of the operators has a backward pass: a result without its gradient would be a silent error."""
    def grad(*s, dtype=torch.float32):
        return torch.zeros(*s, dtype=dtype, requires_grad=True)
    idx, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    pool, new = torch.zeros(5, 2, 16, 64), torch.zeros(2, 2, 64)
    calls = [lambda: paged_attention(**_attn(q=grad(2, 8, 64, dtype=torch.bfloat16))),
             lambda: paged_attention(grad(2, 8, 64), pool, pool, table, idx, k_new=new, v_new=new),
             lambda: paged_attention(torch.zeros(2, 8, 64), pool, pool, table, idx, k_new=new, v_new=grad(2, 2, 64)),
             lambda: paged_write(grad(2, 4, 2, 64), torch.zeros(2, 4, 2, 64), pool, pool, table, idx),
             lambda: copy_pages([pool, grad(5, 3)], idx, idx),
             lambda: beam_reorder(grad(4, 3), table),
             lambda: beam_select(grad(2, 3, 50), torch.zeros(2, 3)),
             lambda: beam_select(torch.zeros(2, 3, 50), grad(2, 3))]
    for call in calls:
        with pytest.raises(ValueError, match="no backward pass"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
            call()


def test_memory_that_would_be_written_twice_is_refused():
    idx, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    one, new = torch.zeros(1, 2, 16, 64), torch.zeros(2, 2, 64)
    with pytest.raises(ValueError, match="expanded"):
        paged_attention(torch.zeros(2, 8, 64), one.expand(5, 2, 16, 64), one.expand(5, 2, 16, 64), table, idx, k_new=new, v_new=new)
    with pytest.raises(ValueError, match="expanded"):
        paged_write(torch.zeros(2, 4, 2, 64), torch.zeros(2, 4, 2, 64), one.expand(5, 2, 16, 64), one.expand(5, 2, 16, 64), table, idx)
    rows = (_cabi.L3Rows * 3)(_cabi.L3Rows(0x1000, 6, 64, 1, 0, 64), _cabi.L3Rows(0x2000, 6, 64, 1, 0, 64), _cabi.L3Rows(0x1000, 6, 64, 1, 0, 64))
    assert _cabi.lib().l3_beam_reorder(0, C.c_void_p(), rows, 3, C.c_void_p(0x1000), 2, 3) == _cabi.L3_EINVAL
    assert b"tensors 0 and 2" in _cabi.lib().l3_last_error(None)


def test_negated_views_are_refused():
    q = torch.zeros(2, 8, 1, dtype=torch.complex64).conj().imag
    assert q.is_neg()
    with pytest.raises(ValueError, match="negated"):
        paged_attention(**_attn(q=q))


def test_rows_are_found():
    """A row as runs of bytes: contiguous, one dimension cut, sequences behind heads."""
    def one(x):
        return _ops().rows(x)
    x = torch.zeros(6, 4, 10, 8)
    assert one(x) == (6, 1280, 1, 0, 1280)
    assert one(x[:, :, 2:5]) == (6, 1280, 4, 320, 96)
    assert one(x[:, 1:3]) == (6, 1280, 1, 0, 640)
    assert one(x.transpose(0, 1)) == (4, 320, 6, 1280, 320)
    assert one(torch.zeros(7)) == (7, 4, 1, 0, 4)
    assert one(torch.zeros(7, 0)) [4] == 0
    assert one(x[:, 0, 0, :1]) == (6, 1280, 1, 0, 4)


def test_c_entries_refuse_before_any_gpu_call():
    lib = _cabi.lib()
    none = C.c_void_p()
    n = C.c_int64()
    assert lib.l3_paged_attention(None) == _cabi.L3_EINVAL
    assert lib.l3_paged_write(None) == _cabi.L3_EINVAL and lib.l3_beam_select(None) == _cabi.L3_EINVAL
    assert lib.l3_paged_attention_workspace(0, 8, 3, 64, C.byref(n)) == _cabi.L3_EINVAL
    assert lib.l3_paged_attention_workspace(0, 8, 2, 40, C.byref(n)) == _cabi.L3_EINVAL
    assert lib.l3_beam_select_workspace(0, 1, 300, 10, 1, C.byref(n)) == _cabi.L3_EINVAL
    assert lib.l3_beam_select_workspace(0, 1, 4, 10, 65, C.byref(n)) == _cabi.L3_EINVAL
    a = _cabi.L3PagedAttention(batch=1, heads=4, kv_heads=2, head_dim=64, pages=4, page_size=12, max_pages=1)
    assert lib.l3_paged_attention(C.byref(a)) == _cabi.L3_EINVAL and b"power of two" in lib.l3_last_error(None)
    a.page_size = 16
    assert lib.l3_paged_attention(C.byref(a)) == _cabi.L3_EINVAL and b"no data" in lib.l3_last_error(None)
    a.max_pages = 1 << 28
    assert lib.l3_paged_attention(C.byref(a)) == _cabi.L3_EINVAL and b"too long" in lib.l3_last_error(None)
    a.max_pages, a.q_dtype = 1, 1
    assert lib.l3_paged_attention(C.byref(a)) == _cabi.L3_EINVAL and b"types" in lib.l3_last_error(None)
    a.q_dtype, a.kv_dtype, a.out_dtype = 0, 0, 0
    a.k.data = a.v.data = 0x1000
    a.k.token_stride = 2
    assert lib.l3_paged_attention(C.byref(a)) == _cabi.L3_EINVAL and b"16 bytes" in lib.l3_last_error(None)
    w = _cabi.L3PagedWrite(batch=70000, tokens=1, kv_heads=2, head_dim=64, pages=4, page_size=16, max_pages=1)
    assert lib.l3_paged_write(C.byref(w)) == _cabi.L3_EINVAL
    rows = (_cabi.L3Rows * 1)(_cabi.L3Rows(0x1000, 6, 64, 1, 0, 64))
    assert lib.l3_beam_reorder(0, none, rows, 1, None, 2, 3) == _cabi.L3_EINVAL
    assert lib.l3_beam_reorder(0, none, rows, 1, C.c_void_p(0x1000), 1, 257) == _cabi.L3_EINVAL
    assert lib.l3_copy_rows(0, none, rows, 1, None, None, 2) == _cabi.L3_EINVAL
    assert lib.l3_copy_rows(0, none, rows, 0, None, None, 0) == _cabi.L3_EINVAL
    s = _cabi.L3BeamSelect(batch=1, beams=2, vocab=10, best=2, eos=10)
    assert lib.l3_beam_select(C.byref(s)) == _cabi.L3_EINVAL and b"eos" in lib.l3_last_error(None)
    s.eos = 3
    assert lib.l3_beam_select(C.byref(s)) == _cabi.L3_EINVAL and b"missing" in lib.l3_last_error(None)


def test_division_by_multiplication():
    """The kernels' x // d for x < 2^31 (d fixed for a launch), as they compute it."""
    import random
    rng = random.Random(1)
    for d in [1, 2, 3, 5, 7, 12, 48, 255, 256, 257, 2048, 4095, 65537, (1 << 30) - 1] + [rng.randrange(1, 1 << 30) for _ in range(200)]:
        sh = 0
        while (1 << sh) < d:
            sh += 1
        mul = ((1 << 32) * ((1 << sh) - d)) // d + 1
        assert mul < 1 << 32
        for x in [0, 1, d - 1, d, d + 1, 2 * d - 1, (1 << 31) - 1] + [rng.randrange(0, 1 << 31) for _ in range(50)]:
            if x < 1 << 31:
                assert (x if sh == 0 else (((x * mul) >> 32) + x) >> sh) == x // d


def test_command_line_end_token_needs_beams():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "generate"), "--model", "nowhere", "--ids", "1", "--eos", "2"], capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 2 and "--beams" in r.stderr
