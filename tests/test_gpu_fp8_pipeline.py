"""GPU: products whose column blocks fill their kernel's ring of stages partly, exactly and
several times over, back to back, so that a CTA starts where another has just left."""
import pytest
import torch

from agent_harness_b200._lib import lib
from test_gpu_fp8 import acts, blocks, fp8  # noqa: F401
from test_gpu_fp8_products import check_product

pytestmark = pytest.mark.gpu

# each kernel: 16, 32 and 64 tokens a CTA, single CTAs, their clusters, pairs
TOKENS = [(1, 700), (20, 700), (50, 700), (100, 20000), (70, 4900), (200, 4000)]


@pytest.mark.parametrize("m,n", TOKENS)
def test_every_number_of_column_blocks(fp8, m, n):  # noqa: F811
    for kb in [1, 2, 3, 4, 5, 6, 7, 8, 9, 11, 12, 13, 15, 16, 17, 24, 25, 33]:
        k = kb * 128 - 5
        wq, ws = blocks(n, k, kb)
        W = fp8.Fp8Weight.from_blocks(wq, ws)
        q, s = acts(fp8, m, k, kb)
        ys = [W.matmul(q, s, dtype=torch.bfloat16) for _ in range(8)]
        check_product(ys[0], q, s, wq, ws)
        assert all(torch.equal(y, ys[0]) for y in ys[1:])
        W.close()
    assert lib().ah_check_device_error(None) == 0


def test_kernels_in_turn(fp8):  # noqa: F811
    """Different kernels after one another on one stream, each starting under the last."""
    work = []
    for m, n in TOKENS:
        wq, ws = blocks(n, 640, m)
        q, s = acts(fp8, m, 640, m)
        work.append((fp8.Fp8Weight.from_blocks(wq, ws), q, s, wq, ws))
    outs = [[W.matmul(q, s) for W, q, s, _, _ in work] for _ in range(20)]
    for i, (W, q, s, wq, ws) in enumerate(work):
        check_product(outs[0][i], q, s, wq, ws)
        assert all(torch.equal(o[i], outs[0][i]) for o in outs)
    assert lib().ah_check_device_error(None) == 0
