"""GPU: many norm rows with few threads each, and batches without rows."""
import pytest
import torch

from test_gpu_fp8 import F, TYPES, fp8, groups, randn  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1000, 1024, 1536, 2048, 2056, 4096])
@pytest.mark.parametrize("m", [297, 700])
def test_norm_of_many_rows(fp8, m, k, dtype):  # noqa: F811
    """More than two rows per SM: as few as 32 threads add a row's squares.  Their sum is off by
    at most (k / 32 + 8 terms of a thread, 10 levels of the tree) 2^-24, half of that after the
    root; mean, eps, root, two quotients, the weight's and the scale's product add 8."""
    x, w = randn(m, k, seed=k, dtype=dtype) * 3, (1 + 0.2 * randn(k, seed=3)).to(dtype)
    r = randn(m, k, seed=k + 1, dtype=dtype)
    tol = ((k / 32 + 18) / 2 + 8) * 2.0**-24
    for res in (None, r):
        h = x.double() if res is None else (x.float() + res.float()).to(dtype).double()
        q, s = fp8.add_rms_norm_fp8(x, w, residual=res)
        if res is not None:
            assert torch.equal(res.double(), h)
        z = h * w.double()
        g, col = groups(z)
        want = g / F / (h.square().mean(1, keepdim=True) + 1e-5).sqrt()
        assert ((s.double() - want).abs() <= tol * want).all()
        v = z * F / col  # h w, 448 / g and their product: 2^-22 covers four roundings
        off = (q.double() - v).abs()
        assert (off <= torch.maximum(v.abs() * 2.0**-4, torch.full_like(v, 2.0**-10)) + 2.0**-22 * v.abs()).all()


@pytest.mark.parametrize("k", [1, 16, 100, 1003, 4096])
def test_no_rows(fp8, k):  # noqa: F811
    """An empty batch is no work at any width, through every row entry and the block."""
    x, w = torch.empty(0, k, device="cuda"), torch.ones(k, device="cuda")
    given = fp8.alloc(0, k)
    for q, s in (fp8.quantize_fp8(x), fp8.swiglu_fp8(x, x), fp8.add_rms_norm_fp8(x, w),
                 fp8.add_rms_norm_fp8(x, w, residual=x.clone()), fp8.quantize_fp8(x, *given)):
        assert q.shape == (0, k) and s.shape == (0, (k + 127) // 128)
    W = fp8.Fp8Weight.from_float(randn(70, k))
    assert W.matmul(*given).shape == (0, 70)
    block = fp8.Fp8SwigluBlock.from_float(randn(70, k), randn(70, k), randn(k, 70))
    assert block(x, w, residual=x.clone()).shape == (0, k)
