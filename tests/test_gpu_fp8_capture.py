"""GPU: a weight is not made under capture, and the attempt leaves the capture whole."""
import pytest
import torch

from agent_harness_b200._lib import AhError
from test_gpu_fp8 import blocks, fp8, randn  # noqa: F401

pytestmark = pytest.mark.gpu


def test_makers_refuse_a_capturing_stream(fp8):  # noqa: F811
    w = randn(256, 256)
    wq, ws = blocks(256, 256, 1)
    W = fp8.Fp8Weight.from_float(w)
    q, s = fp8.quantize_fp8(randn(4, 256, seed=2))
    y = torch.zeros(4, 256, device="cuda")
    want = W.matmul(q, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for make in (lambda: fp8.Fp8Weight.from_float(w), lambda: fp8.Fp8Weight.from_blocks(wq, ws),
                     lambda: fp8.Fp8SwigluBlock.from_float(w, w, w)):
            with pytest.raises(AhError) as e:
                make()
            assert e.value.status == -1 and "captur" in str(e.value)
        W.matmul(q, s, out=y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_a_weight_may_go_during_a_capture(fp8):  # noqa: F811
    """Closed, or collected, while its thread captures something else: it is freed, and the
    capture goes on."""
    W, old = fp8.Fp8Weight.from_float(randn(256, 256)), fp8.Fp8Weight.from_float(randn(16384, 16384))
    q, s = fp8.quantize_fp8(randn(4, 256, seed=2))
    want, y = W.matmul(q, s), torch.zeros(4, 256, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        old.close()
        W.matmul(q, s, out=y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    assert torch.cuda.mem_get_info()[0] > free + 200 * 2**20  # 256 MB less what the capture took
