"""GPU suite: rows of a rotary call that stay as they are, bit for bit."""
import math

import pytest
import torch

from llama3_np_b200 import paged_rotary_write, rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def odd_rows(rows, heads, dim, dtype, seed):
    """Ordinary numbers beside infinities, NaN, both zeros and the type's largest and smallest."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, heads, dim, generator=g, device="cuda").to(dtype)
    info = torch.finfo(dtype)
    special = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0, info.max, info.min, info.tiny, info.smallest_normal / 4], device="cuda").to(dtype)
    pick = torch.randint(0, 30, x.shape, generator=g, device="cuda")
    return torch.where(pick < len(special), special[pick.clamp(max=len(special) - 1)], x)


def bits(x):
    return x.contiguous().view(torch.int32 if x.dtype == torch.float32 else torch.int16)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("dim,dims", [(128, 128), (96, 24), (6, 6), (10, 2)])
@pytest.mark.parametrize("rows", [5, 1001])
@pytest.mark.parametrize("inverse", [False, True])
def test_rows_at_negative_positions_stay(kind, layout, dim, dims, rows, inverse):
    x = odd_rows(rows, 3, dim, TYPES[kind], rows + dim)
    positions = torch.arange(rows, dtype=torch.int32, device="cuda") + 7
    positions[::3], positions[1::6] = -1, -2 ** 31
    f, _ = rotary_frequencies(dims)
    got = rotary(x, positions, f, layout=layout, amplitude=1.5, inverse=inverse)
    stay = positions < 0
    assert torch.equal(bits(got[stay]), bits(x[stay])) and torch.equal(bits(got[..., dims:]), bits(x[..., dims:]))
    # the others: the formula in 64 bits on every pair of numbers (two products and a sum in fp32, the angle's rounding, the result's)
    a, b = (x[..., :dims:2], x[..., 1:dims:2]) if layout == "pairs" else (x[..., :dims // 2], x[..., dims // 2:dims])
    c, d = (got[..., :dims:2], got[..., 1:dims:2]) if layout == "pairs" else (got[..., :dims // 2], got[..., dims // 2:dims])
    angle = (positions.double()[:, None] * f)[:, None] * (-1 if inverse else 1)
    fine = (a.isfinite() & b.isfinite() & (a.abs() < 1e4) & (b.abs() < 1e4) & ~stay[:, None, None])
    for have, want in ((c, 1.5 * (a.double() * angle.cos() - b.double() * angle.sin())), (d, 1.5 * (b.double() * angle.cos() + a.double() * angle.sin()))):
        bound = 1.5 * (a.double().abs() + b.double().abs()) * 2.0 ** -21 + want.abs() * torch.finfo(TYPES[kind]).eps / 2 + torch.finfo(TYPES[kind]).smallest_normal
        assert bool(((have.double() - want).abs() <= bound)[fine].all()) and int(fine.sum()) > 0
    own = x.clone()
    assert rotary(own, positions, f, layout=layout, amplitude=1.5, inverse=inverse, out=own) is own and torch.equal(bits(own), bits(got))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_keys_at_negative_positions_are_written_as_they_are(kind, layout):
    """A slot without a position: the key goes there unturned, the value as ever."""
    dtype, rows = TYPES[kind], 40
    q, k, v = odd_rows(rows, 4, 64, dtype, 1), odd_rows(rows, 2, 64, dtype, 2), odd_rows(rows, 2, 64, dtype, 3)
    pools = [torch.zeros(4, 2, 16, 64, dtype=dtype, device="cuda") for _ in range(2)]
    slots = torch.randperm(64, generator=torch.Generator().manual_seed(4))[:rows].cuda()
    positions = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    got = paged_rotary_write(q, k, v, positions, slots, *pools, rotary_frequencies(64)[0], layout=layout)
    assert torch.equal(bits(got), bits(q))
    for x, pool in ((k, pools[0]), (v, pools[1])):
        assert torch.equal(bits(pool.transpose(1, 2).reshape(64, 2, 64)[slots]), bits(x))
