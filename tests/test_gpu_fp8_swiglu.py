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


@pytest.mark.parametrize("m,n_embd,n_ff", [(1, 512, 1100), (20, 256, 700), (130, 384, 700), (100, 256, 12900), (400, 700, 2500), (320, 8192, 2000)])
def test_block_with_far_gates(fp8, m, n_embd, n_ff):  # noqa: F811
    """Every kernel of the block: gates of about -30, -86, -88, -89, -110 and -150 by tiles of
    128, ups of 1e25 and more, and outputs that see one tile each.  Against the block's
    steps: the activations may sit one e4m3 step (2^-3) apart where a last bit differs."""
    tiles, kb = (n_ff + 127) // 128, (n_embd + 127) // 128
    x = 1 + 0.1 * randn(m, n_embd, seed=1).clamp(-2, 2)  # normalised: about 1 everywhere
    w = torch.ones(n_embd, device="cuda")
    gate = torch.tensor([-30.0, -86.2, -88.0, -89.0, -110.0, -150.0], device="cuda")[torch.arange(tiles, device="cuda") % 6]
    gq = torch.full((n_ff, n_embd), 1.0, device="cuda").to(torch.float8_e4m3fn)
    gs = (gate / n_embd)[:, None].repeat(1, kb)
    uq = randn(n_ff, n_embd, seed=2).clamp(-4, 4).to(torch.float8_e4m3fn)
    us = torch.full((tiles, kb), 1e25, device="cuda") * torch.exp2(torch.arange(tiles, device="cuda") % 6 * 4.0)[:, None]
    tile_of = torch.arange(n_embd, device="cuda")[:, None] % tiles == torch.arange(n_ff, device="cuda")[None] // 128
    dq = (randn(n_embd, n_ff, seed=3).clamp(-4, 4) * tile_of).to(torch.float8_e4m3fn)
    ds = torch.full((kb, tiles), 2.0**-4, device="cuda")
    block = fp8.Fp8SwigluBlock.from_blocks(gq, gs, uq, us, dq, ds)
    y = block(x, w)
    q, s = fp8.add_rms_norm_fp8(x, w)
    gu = block.gate_up.matmul(q, s)
    assert (gu[:, :n_ff] < -25).all() and (gu[:, :n_ff].amin() < -100 if tiles > 4 else True)
    a, asc = fp8.swiglu_fp8(gu[:, :n_ff], gu[:, n_ff:])
    check(a, asc, swiglu(gu[:, :n_ff], gu[:, n_ff:]))
    want = block.down.matmul(a, asc)
    seen = (torch.arange(n_embd, device="cuda") % tiles) % 6 != 5  # -150: below the smallest group's scale
    assert torch.isfinite(y).all()
    step = a.float().abs().clamp(min=2.0**-6) * 2.0**-3 * asc.repeat_interleave(G, 1)[:, :n_ff]
    bound = step.double() @ (dq.double().abs() * 2.0**-4).t() + 2.0**-16 * want.abs().double() + 1e-30
    assert ((y.double() - want.double()).abs() <= bound).all()
    assert (y[:, seen].double() - want[:, seen]).norm() <= 2.0**-8 * want[:, seen].norm()
    per_tile = y.abs().amax(0)
    assert (per_tile[seen] > 0).all()
    block.close()
