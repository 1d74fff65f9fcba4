"""CPU suite: what the operators of a packed step refuse, from Python and through the C-ABI, and the frequencies of rotary positions."""
import ctypes as C
import math

import pytest
import torch

from llama3_np_b200 import (_cabi, paged_chunk_attention, paged_extend, paged_rotary_write, rotary, rotary_frequencies, token_logprobs)


def ints(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


def _extend(**change):
    a = dict(page_table=ints(3, 4), lengths=ints(3), counts=ints(3), free_pages=ints(5), page_size=16, tokens=7)
    a.update(change)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(page_table=ints(2, 4)), "rows"), (dict(page_table=ints(3, 4, dtype=torch.int64)), "type"), (dict(page_table=ints(4, 3).T), "contiguous"),
    (dict(page_table=ints(1, 4).expand(3, 4)), "expanded"), (dict(lengths=ints(3, 1)), "dimensions"), (dict(lengths=ints(6)[::2]), "contiguous"),
    (dict(counts=ints(2)), "counts"), (dict(counts=ints(3, dtype=torch.int64)), "type"), (dict(free_pages=ints(5, dtype=torch.int64)), "type"),
    (dict(free_pages=ints(10)[::2]), "contiguous"), (dict(page_size=12), "power of two"), (dict(page_size=0), "power of two"),
    (dict(page_size=1 << 17), "power of two"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 31), "too large"), (dict(lengths=[1, 2, 3]), "tensor"),
    (dict(), "CUDA device"),
])
def test_extend_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        paged_extend(**_extend(**change))


def test_numbers_that_are_none_raise_a_type_error():
    with pytest.raises(TypeError):
        paged_extend(**_extend(tokens="7"))
    with pytest.raises(TypeError):
        token_logprobs(torch.zeros(2, 9), ints(2), top=1.5)


def _chunk(dtype=torch.bfloat16, **change):
    a = dict(q=torch.zeros(7, 8, 64, dtype=dtype), k_pages=torch.zeros(5, 2, 16, 64, dtype=dtype), v_pages=torch.zeros(5, 2, 16, 64, dtype=dtype),
             page_table=ints(3, 4), lengths=ints(3), starts=ints(4))
    a.update(change)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(8, 64, dtype=torch.bfloat16)), "dimensions"), (dict(q=torch.zeros(7, 8, 64)), "type"),
    (dict(q=torch.zeros(7, 9, 64, dtype=torch.bfloat16)), "heads over"), (dict(q=torch.zeros(7, 8, 32, dtype=torch.bfloat16)), "head size"),
    (dict(q=torch.zeros(7, 64, 8, dtype=torch.bfloat16).transpose(1, 2)), "contiguous"),
    (dict(q=torch.zeros(7, 8, 68, dtype=torch.bfloat16)[..., 4:]), "16 bytes"),
    (dict(v_pages=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)), "differ"), (dict(lengths=ints(2)), "rows"), (dict(starts=ints(3)), "starts"),
    (dict(starts=ints(4, dtype=torch.int64)), "type"), (dict(starts=ints(8)[::2]), "contiguous"), (dict(page_table=ints(4, 3).T), "contiguous"),
    (dict(out=torch.zeros(7, 8, 64)), "type"), (dict(out=torch.zeros(7, 8, 128, dtype=torch.bfloat16)[..., :64]), "out"), (dict(), "CUDA device"),
])
def test_chunk_attention_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        paged_chunk_attention(**_chunk(**change))


def test_chunk_attention_refuses_its_own_query_as_out():
    a = _chunk()
    with pytest.raises(ValueError, match="shares memory"):
        paged_chunk_attention(**a, out=a["q"])


@pytest.mark.parametrize("args,kw,text", [
    ((torch.zeros(7, 64), ints(7)), {}, r"\[tokens, heads, size\]"), ((torch.zeros(7, 2, 64).double(), ints(7)), {}, "type"),
    ((torch.zeros(7, 2, 64), ints(6)), {}, "positions"), ((torch.zeros(7, 2, 64), ints(7, dtype=torch.int64)), {}, "type"),
    ((torch.zeros(2, 7, 2, 64), ints(14)), {}, "positions"), ((torch.zeros(2, 7, 2, 64), ints(7, 2).T), {}, "contiguous"),
    ((torch.zeros(7, 2, 64), ints(7)), {"layout": "rows"}, "layout"), ((torch.zeros(7, 2, 64), ints(7)), {"layout": 1}, "layout"),
    ((torch.zeros(7, 2, 16), ints(7)), {}, "frequencies"), ((torch.zeros(7, 64, 2).transpose(1, 2), ints(7)), {}, "contiguous"),
    ((torch.zeros(7, 2, 64), ints(7)), {"out": torch.zeros(7, 2, 64).half()}, "type"), ((torch.zeros(7, 2, 64), ints(7)), {"out": torch.zeros(7, 2, 32)}, "out"),
    ((torch.zeros(7, 2, 64), ints(7)), {"out": torch.zeros(7, 1, 64).expand(7, 2, 64)}, "expanded"),
    ((torch.zeros(7, 2, 1100), ints(7)), {}, "up to 1024"), ((torch.zeros(7, 2, 64), ints(7)), {}, "CUDA device"),
])
def test_rotary_refuses(args, kw, text):
    with pytest.raises(ValueError, match=text):
        rotary(*args, torch.zeros(16, dtype=torch.float64), **kw)


def test_rotary_refuses_what_shares_memory_and_odd_frequencies():
    x = torch.zeros(9, 2, 64)
    f = torch.zeros(16, dtype=torch.float64)
    with pytest.raises(ValueError, match="shares memory"):
        rotary(x[1:], ints(8), f, out=x[:-1])
    with pytest.raises(ValueError, match="CUDA device"):
        rotary(x, ints(9), f, out=x)
    for bad, text in [(f.float(), "type"), (f[::2], "contiguous"), (f[None], "dimensions")]:
        with pytest.raises(ValueError, match=text):
            rotary(x, ints(9), bad)


def _write(**change):
    a = dict(q=torch.zeros(7, 8, 64), k=torch.zeros(7, 2, 64), v=torch.zeros(7, 2, 64), positions=ints(7), slots=ints(7, dtype=torch.int64),
             k_pages=torch.zeros(5, 2, 16, 64), v_pages=torch.zeros(5, 2, 16, 64), frequencies=torch.zeros(32, dtype=torch.float64))
    a.update(change)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(7, 8, 32)), "q must be"), (dict(q=torch.zeros(7, 8, 64).half()), "type"), (dict(k=torch.zeros(6, 2, 64)), "k must be"),
    (dict(v=torch.zeros(7, 3, 64)), "v must be"), (dict(k=torch.zeros(7, 64, 2).transpose(1, 2)), "contiguous"), (dict(positions=ints(6)), "positions"),
    (dict(slots=ints(7)), "type"), (dict(slots=ints(6, dtype=torch.int64)), "slots"), (dict(k_pages=torch.zeros(5, 2, 12, 64), v_pages=torch.zeros(5, 2, 12, 64)), "power of two"),
    (dict(k_pages=torch.zeros(1, 2, 16, 64).expand(5, 2, 16, 64)), "expanded"), (dict(frequencies=torch.zeros(33, dtype=torch.float64)), "frequencies"),
    (dict(out=torch.zeros(7, 8, 32)), "out"), (dict(layout="x"), "layout"), (dict(), "CUDA device"),
])
def test_rotary_write_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        paged_rotary_write(**_write(**change))


def test_rotary_write_refuses_results_over_what_it_reads():
    qkv = torch.zeros(7, 12, 64)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    for a, out in [(_write(k=torch.zeros(7, 8, 64)[:, :2]), "k"), (_write(v=torch.zeros(7, 8, 64)[:, :2]), "v"), (_write(), "q")]:
        with pytest.raises(ValueError, match="shares memory"):
            paged_rotary_write(**a, out=a[out].as_strided((7, 8, 64), (512, 64, 1)) if out != "q" else a["q"].as_strided((7, 8, 64), (64, 448, 1)))
    with pytest.raises(ValueError, match="CUDA device"):   # q itself, beside k and v in one tensor
        paged_rotary_write(**_write(q=q, k=k, v=v), out=q)


@pytest.mark.parametrize("args,kw,text", [
    ((torch.zeros(9), ints(1)), {}, "dimensions"), ((torch.zeros(2, 9).double(), ints(2)), {}, "type"), ((torch.zeros(2, 9), ints(3)), {}, "tokens"),
    ((torch.zeros(2, 9), ints(2, dtype=torch.int64)), {}, "type"), ((torch.zeros(9, 2).T, ints(2)), {}, "contiguous"),
    ((torch.zeros(2, 99), ints(2)), {"top": 65}, "top"), ((torch.zeros(2, 9), ints(2)), {"top": 10}, "top"), ((torch.zeros(2, 9), ints(2)), {"top": -1}, "top"),
    ((torch.zeros(2, 0), ints(2)), {}, "tokens"), ((torch.zeros(2, 9), ints(2)), {}, "CUDA device"),
])
def test_logprobs_refuses(args, kw, text):
    with pytest.raises(ValueError, match=text):
        token_logprobs(*args, **kw)


def test_gradients_are_refused():
    def grad(x):
        return x.clone().requires_grad_()
    calls = [lambda: paged_chunk_attention(**_chunk(q=grad(torch.zeros(7, 8, 64, dtype=torch.bfloat16)))),
             lambda: rotary(grad(torch.zeros(7, 2, 64)), ints(7), torch.zeros(16, dtype=torch.float64)),
             lambda: rotary(torch.zeros(7, 2, 64), ints(7), grad(torch.zeros(16, dtype=torch.float64))),
             lambda: paged_rotary_write(**_write(v=grad(torch.zeros(7, 2, 64)))),
             lambda: token_logprobs(grad(torch.zeros(2, 9)), ints(2))]
    for call in calls:
        with pytest.raises(ValueError, match="no backward pass"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
            call()


def test_c_entries_refuse_before_any_gpu_call():
    lib, n = _cabi.lib(), C.c_int64()

    def refuses(rc, text):
        assert rc == _cabi.L3_EINVAL and text in lib.l3_last_error(None), lib.l3_last_error(None)
    for call in (lib.l3_paged_extend, lib.l3_rotary, lib.l3_paged_chunk_attention, lib.l3_token_logprobs):
        refuses(call(None), b"no arguments")
    e = _cabi.L3PagedExtend(batch=1, tokens=1, max_pages=1, page_size=3)
    refuses(lib.l3_paged_extend(C.byref(e)), b"power of two")
    e.page_size = 4
    refuses(lib.l3_paged_extend(C.byref(e)), b"missing")
    e.batch = -1
    refuses(lib.l3_paged_extend(C.byref(e)), b"bad sizes")
    r = _cabi.L3Rotary(batch=1, tokens=1, heads=1, head_dim=8, dims=7)
    refuses(lib.l3_rotary(C.byref(r)), b"even number")
    r.dims = 10
    refuses(lib.l3_rotary(C.byref(r)), b"even number")
    r.dims, r.layout = 8, 2
    refuses(lib.l3_rotary(C.byref(r)), b"layout")
    r.layout = 0
    refuses(lib.l3_rotary(C.byref(r)), b"missing")
    r.kv_heads, r.batch = 1, 2
    refuses(lib.l3_rotary(C.byref(r)), b"one batch")
    refuses(lib.l3_paged_chunk_workspace(0, 1, 8, 3, 64, 0, C.byref(n)), b"multiple")
    refuses(lib.l3_paged_chunk_workspace(0, 1, 8, 2, 40, 0, C.byref(n)), b"unsupported")
    refuses(lib.l3_paged_chunk_workspace(0, 1, 8, 2, 64, 9, C.byref(n)), b"dtype")
    refuses(lib.l3_paged_chunk_workspace(0, 1 << 30, 8, 2, 64, 0, C.byref(n)), b"too many")
    c = _cabi.L3PagedChunk(batch=1, tokens=1, heads=2, kv_heads=1, head_dim=64, pages=1, page_size=6, max_pages=1)
    refuses(lib.l3_paged_chunk_attention(C.byref(c)), b"power of two")
    c.page_size = 8
    refuses(lib.l3_paged_chunk_attention(C.byref(c)), b"no data")
    c.k.data = c.v.data = 0x1008
    refuses(lib.l3_paged_chunk_attention(C.byref(c)), b"16 bytes")
    c.k.data = c.v.data = 0x1000
    refuses(lib.l3_paged_chunk_attention(C.byref(c)), b"missing")
    t = _cabi.L3TokenLogprobs(rows=1, vocab=9, top=10)
    refuses(lib.l3_token_logprobs(C.byref(t)), b"top")
    t.top = 65
    refuses(lib.l3_token_logprobs(C.byref(t)), b"top")
    t.top, t.vocab = 0, 1 << 24
    refuses(lib.l3_token_logprobs(C.byref(t)), b"vocab")
    t.vocab = 9
    refuses(lib.l3_token_logprobs(C.byref(t)), b"missing")


def test_frequencies():
    plain, one = rotary_frequencies(8, 100.0, device="cpu")
    assert one == 1.0 and plain.dtype == torch.float64
    assert torch.allclose(plain, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(rotary_frequencies(8, 100.0, kind="linear", factor=4.0, device="cpu")[0], plain / 4, rtol=1e-15)
    ntk = rotary_frequencies(8, 100.0, kind="ntk", factor=4.0, device="cpu")[0]
    assert math.isclose(ntk[0], 1.0) and math.isclose(ntk[3], plain[3] / 4, rel_tol=1e-14)
    # 5000 positions: turns 795.8, 251.6, 79.6, 25.2
    f = rotary_frequencies(8, 100.0, kind="llama3", factor=8.0, original=5000, low=50.0, high=100.0, device="cpu")[0]
    fade = (5000 * 0.1 / (2 * math.pi) - 50) / 50
    want = [1.0, 100 ** -0.25, 0.1 * (fade + (1 - fade) / 8), 100 ** -0.75 / 8]
    assert torch.allclose(f, torch.tensor(want, dtype=torch.float64), rtol=1e-14)
    f, a = rotary_frequencies(64, 10000.0, kind="yarn", factor=16.0, original=4096, low=1.0, high=32.0, device="cpu")
    plain = rotary_frequencies(64, 10000.0, device="cpu")[0]
    turns = 4096 * plain / (2 * math.pi)
    assert math.isclose(a, 0.1 * math.log(16) + 1)
    pair = 64 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000))          # the pair of 32 turns
    last = 64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000))               # of one
    assert torch.equal(f[turns >= 40], plain[turns >= 40]) and torch.allclose(f[turns < 0.7], plain[turns < 0.7] / 16, rtol=1e-15)
    i = 16
    assert math.floor(pair) < i < math.ceil(last)
    keep = 1 - (i - math.floor(pair)) / (math.ceil(last) - math.floor(pair))
    assert math.isclose(f[i], plain[i] * (keep + (1 - keep) / 16), rel_tol=1e-13)


@pytest.mark.parametrize("args,kw", [((7,), {}), ((0,), {}), ((8.0,), {}), ((8, 0.0), {}), ((8, math.inf), {}), ((8,), {"kind": "x"}), ((8,), {"kind": "linear", "factor": 0.5}),
                                     ((2,), {"kind": "ntk", "factor": 2.0}), ((8,), {"kind": "llama3", "low": 4.0, "high": 4.0}),
                                     ((8,), {"kind": "yarn", "original": 0}), ((8, 1.0), {"kind": "yarn", "high": 32.0})])
def test_frequencies_refuse(args, kw):
    with pytest.raises(ValueError):
        rotary_frequencies(*args, device="cpu", **kw)
