"""GPU: e4m3 products against the 64-bit formula with a check that a NaN, or any value
that does not compare, fails; outputs and weights of more than 2^31 elements.

Tolerance, as for every product here: sums of 128 exact terms per block and then over
the blocks are off by at most (128 + blocks + 4) 2^-23 of the sum of magnitudes (2^-23:
the tensor cores may truncate), and the output's rounding by eps / 2 (an f16 subnormal's
by 2^-25)."""
import pytest
import torch

from test_gpu_fp8 import G, LARGE, SHAPES, SPLIT, TYPES, WHOLE, acts, block_spread, blocks, fp8, spread  # noqa: F401


def check_near(y, want, tol):
    """|y - want| <= tol everywhere; a NaN in y is never near."""
    ok = (y.double() - want).abs() <= tol
    assert ok.all(), ((~ok).nonzero()[:4].tolist(), int((~ok).sum()))


def check_product(y, q, s, wq, ws):
    a, w = q.double() * spread(s, q.shape), wq.double() * block_spread(ws, wq.shape)
    want, mag = a @ w.t(), a.abs() @ w.abs().t()
    tol = (G + (q.shape[1] + G - 1) // G + 4) * 2.0**-23 * mag + want.abs() * torch.finfo(y.dtype).eps / 2 * 1.001
    check_near(y, want, tol + (2.0**-25 if y.dtype == torch.float16 else 0.0))


def test_the_check_sees_a_nan():
    """CPU: one NaN among right values fails the check."""
    want = torch.ones(3, 4, dtype=torch.float64)
    y = want.float()
    check_near(y, want, torch.full_like(want, 1e-9))
    y[1, 2] = float("nan")
    with pytest.raises(AssertionError):
        check_near(y, want, torch.full_like(want, 1e-9))
    with pytest.raises(AssertionError):
        check_near(y, want, torch.full_like(want, float("inf")))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES + LARGE + SPLIT + WHOLE)
def test_products(fp8, m, n, k):  # noqa: F811
    wq, ws = blocks(n, k, m + n + k)
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    q, s = acts(fp8, m, k, 1)
    for dtype in TYPES:
        check_product(W.matmul(q, s, dtype=dtype), q, s, wq, ws)
    W.close()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 300), (3, 300), (20, 300), (40, 300), (100, 20000), (100, 4864), (260, 300), (900, 1500)])
def test_poison_around_the_inputs(fp8, m, n):  # noqa: F811
    """NaN bytes past the activations' columns and rows, NaN scales around the live ones, outputs
    inside a larger matrix: nothing of it arrives, in every kernel."""
    k = 500 if n != 4864 else 1250
    wq, ws = blocks(n, k + 3, 5)
    wq = wq[:, 1:k + 1]
    kb = (k + G - 1) // G
    ws = ws[:, :kb]
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    q0, s0 = acts(fp8, m, k, 2)
    q = torch.full((m + 1, (k + 31) // 16 * 16), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    q[:m, :k].copy_(q0)
    s = torch.full((m + 1, kb + 5), float("nan"), device="cuda")
    s[:m, 2:2 + kb] = s0
    for off, dtype in ((0, torch.float32), (1, torch.float32), (8, torch.bfloat16), (3, torch.float16)):
        y = torch.full((m + 2, n + 24), -3.0, dtype=dtype, device="cuda")
        out = y[1:m + 1, off:off + n]
        W.matmul(q[:m, :k], s[:m, 2:2 + kb], out=out)
        check_product(out, q0, s0, wq, ws)
        assert (y[0] == -3).all() and (y[m + 1] == -3).all()
        assert (y[:, :off] == -3).all() and (y[:, off + n:] == -3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 20, 50, 100, 300, 1648])
@pytest.mark.parametrize("n", [1497, 1498, 1499, 1500, 1501, 1502, 1503, 20001])
def test_neighbours_of_ragged_outputs(fp8, m, n):  # noqa: F811
    """Rows that end inside a 16-byte piece of a wider matrix whose rows start at such
    pieces: the rest of the piece belongs to someone else."""
    wq, ws = blocks(n, 160, 3)
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    q, s = acts(fp8, m, 160, 2)
    for dtype in TYPES:
        y = torch.full((m + 2, (n + 15) // 8 * 8 + 8), -3.0, dtype=dtype, device="cuda")
        W.matmul(q, s, out=y[:m, :n])
        assert (y[:, n:] == -3).all() and (y[m:] == -3).all()
        check_product(y[:m, :n], q, s, wq, ws)


# 16800 tokens over a vocabulary of 128256: 2^31 elements end inside row 16744.  128 tokens
# over 16.8 million rows: output and weight pass 2^31 elements.
HUGE = [(16800, 128256, 128, 128256), (16800, 128256, 128, 128257), (128, 16800000, 128, 16800000)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,ldy", HUGE)
def test_more_elements_than_31_bits(fp8, m, n, k, ldy):  # noqa: F811
    g = torch.Generator("cuda").manual_seed(m)
    w8 = torch.randint(0, 0x70, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    wq, ws = w8.view(torch.float8_e4m3fn), torch.rand((n + G - 1) // G, 1, generator=g, device="cuda") + 0.5
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    q, s = acts(fp8, m, k, 2)
    y = torch.empty(m, ldy, dtype=torch.bfloat16, device="cuda")[:, :n]
    W.matmul(q, s, out=y)
    border = 2**31 // ldy
    rows = torch.tensor(sorted({0, 1, m // 2, m - 1, *(min(border + i, m - 1) for i in (-1, 0, 1))}), device="cuda")
    cols = n - n % G - 10 * G
    for at in (slice(0, 300), slice(cols, n)):
        first = at.start // G
        check_product(y[rows][:, at], q[rows], s[rows], wq[at], ws[first:first + (at.stop - at.start + G - 1) // G])
    for at in range(0, n, 1 << 20):  # no value was left out
        assert torch.isfinite(y[:, at:at + (1 << 20)]).all()
    W.close()
