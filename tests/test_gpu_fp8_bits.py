"""GPU: the quantiser's bits.  q = e4m3(z (448 / g)) and scale = g (1 / 448), each quotient
and product rounded once to f32: the same steps on the CPU, whose division is correctly
rounded, give the same bits.  Most values lie within three f32 steps of the border between
two e4m3 numbers, so that a quotient 448 / g that is off by its last bit shows."""
import pytest
import torch

from test_gpu_fp8 import F, G, TINY, fp8  # noqa: F401

pytestmark = pytest.mark.gpu


def borders():
    v = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    return (v[1:] + v[:-1]) / 2


def expected(x):
    g = x.view(x.shape[0], -1, G).abs().amax(2).clamp(min=TINY)
    v = x.view(x.shape[0], -1, G) * (torch.tensor(F) / g)[:, :, None]
    return v.view_as(x).to(torch.float8_e4m3fn), g * torch.tensor(1 / F, dtype=torch.float32)


@pytest.mark.parametrize("low,high", [(-100, -60), (-60, 0), (-1, 1), (0, 60), (60, 128)])
def test_bits_at_the_borders(fp8, low, high):  # noqa: F811
    rng = torch.Generator().manual_seed(low)
    rows, groups = 512, 16
    g = torch.exp2(low + (high - low) * torch.rand(rows, groups, generator=rng, dtype=torch.float64)).float()
    g = g.clamp(min=TINY, max=torch.finfo(torch.float32).max)
    if low == -1:  # every kind of mantissa: ends, all ones, powers of two
        g.view(-1)[:4096] = (0x3F800000 + torch.arange(4096, dtype=torch.int32) * 2048 + torch.arange(4096, dtype=torch.int32) % 3 - 1).view(torch.float32)
    b = borders()[torch.randint(0, 126, (rows, groups, G), generator=rng)]
    x = (b * g[:, :, None].double() / F).float()
    x = (x.view(torch.int32) + torch.randint(-3, 4, x.shape, generator=rng, dtype=torch.int32)).view(torch.float32)
    x = torch.minimum(x, g[:, :, None]) * torch.where(torch.rand(x.shape, generator=rng) < 0.5, -1.0, 1.0)
    x[:, :, 5] = g
    x = x.view(rows, groups * G)
    q, s = fp8.quantize_fp8(x.cuda())
    wq, ws = expected(x)
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu().view(torch.uint8), wq.view(torch.uint8))


def test_bits_of_ordinary_rows(fp8):  # noqa: F811
    rng = torch.Generator().manual_seed(1)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = torch.randn(300, 2048, generator=rng).to(dtype)
        q, s = fp8.quantize_fp8(x.cuda())
        wq, ws = expected(x.float())
        assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu().view(torch.uint8), wq.view(torch.uint8))
