"""GPU: SwiGLU over the whole range of gates, where exp(-gate) passes the largest f32 too.

Tolerance, in units of 2^-24: the exponential is off by 4 (2^x, documented as 2^-22), by 4
more (ln 2's constant, up to 86) or by a second 2^x and its product, 5 (below -86), by a
rounding for its factor and one for 1 + it, the reciprocal by 2, two products by 1 each: 15.
A value against its group's maximum has that error twice, and two roundings more: 2^-19
covers 32 of them.
Below a gate of -173.9 a value is under 2^-115 whatever up is and may come out as 0."""
import pytest
import torch

from test_gpu_fp8 import F, G, TYPES, fp8, groups, randn  # noqa: F401

pytestmark = pytest.mark.gpu
SLACK = 2.0**-19


def swiglu(gate, up):
    """In 64 bits, without the overflow of exp(-gate)."""
    g, u = gate.double(), up.double()
    e = torch.exp(-g.abs())
    return g * torch.where(g < 0, e, 1.0) / (1 + e) * u


def check(q, s, z):
    g, col = groups(z)
    assert ((s.double() - g / F).abs() <= SLACK * g / F).all()
    v = z * F / col
    off = (q.double() - v).abs()
    assert (off <= torch.maximum(v.abs() * 2.0**-4, torch.full_like(v, 2.0**-10)) + SLACK * v.abs()).all()


def rows(dtype, gates, up_scale):
    """A row per gate, whose groups hold it and its neighbours in the type."""
    g = torch.tensor(gates, device="cuda", dtype=torch.float64)[:, None] * (1 + 0.002 * torch.rand(len(gates), 300, device="cuda", dtype=torch.float64))
    return g.to(dtype), (randn(len(gates), 300, seed=7).clamp(-1, 1).double() * up_scale).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_gate(fp8, dtype):  # noqa: F811
    gates = [-170 + 0.25 * i for i in range(1000)]
    big = 60000.0 if dtype == torch.float16 else 3e38
    for scale in (1.0, big):
        live = [g for g in gates if scale == 1.0 or g < -4]  # gate * up stays below the largest f32
        gate, up = rows(dtype, live, scale)
        check(*fp8.swiglu_fp8(gate, up), swiglu(gate, up))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_around_the_largest_exponential(fp8, dtype):  # noqa: F811
    """exp(-gate) leaves f32 at -88.72, its reciprocal leaves the normal numbers at -87.34."""
    gate, up = rows(dtype, [-89 + 0.01 * i for i in range(301)], 3e38)
    z = swiglu(gate, up)
    assert (z.abs().amax(1) > 1).all()
    check(*fp8.swiglu_fp8(gate, up), z)


@pytest.mark.parametrize("dtype", TYPES)
def test_huge_gates(fp8, dtype):  # noqa: F811
    """Far below, the product is 0; far above, the gate itself."""
    top = torch.finfo(dtype).max
    gate = torch.full((2, 200), -top, dtype=dtype, device="cuda")
    gate[1] = top
    gate[:, 100:] /= 64
    up = torch.full((2, 200), 2.0**-7, dtype=dtype, device="cuda")
    q, s = fp8.swiglu_fp8(gate, up)
    assert (q[0].float() == 0).all() and torch.isfinite(s).all()
    check(q[1:], s[1:], gate[1:].double() * up[1:].double())
    # every finite gate gives a finite product with a small up
    x = (torch.randn(64, 1000, device="cuda", dtype=torch.float64) * 8).exp2().exp2().clamp(max=top)
    x = (x * torch.where(torch.rand_like(x) < 0.5, -1.0, 1.0)).to(dtype)
    q, s = fp8.swiglu_fp8(x, torch.full_like(x, 2.0**-9))
    assert torch.isfinite(s).all() and torch.isfinite(q.float()).all()
