"""CPU: the 8-bit floating point front-end's own rules, on tensors without a device."""
import pytest
import torch

from agent_harness_b200 import fp8
from agent_harness_b200._lib import AhError

CPU = -1  # what Tensor.get_device() gives


@pytest.mark.parametrize("k", [1, 16, 100, 1003])
@pytest.mark.parametrize("m", [0, 1, 3])
def test_row_strides_of_any_batch(m, k):
    """alloc's pairs pass their own check with a row stride of whole 16-byte pieces; torch
    calls a matrix of one row or none contiguous, whatever its stride."""
    ldq, lds = fp8._quantised(*fp8.alloc(m, k, "cpu"), m, k, CPU)
    assert ldq == (k + 15) // 16 * 16 and lds == (k + 127) // 128


@pytest.mark.parametrize("shapes", [((8,), (8,), (8,)), ((), (), ()), ((4, 8), (4, 8), (8,)), ((2, 4, 8), (2, 4, 8), (4, 2)),
                                    ((4, 8), (4, 8), (8, 5)), ((4, 8), (4, 9), (8, 4))])
def test_blocks_of_no_matrices_are_refused(shapes):
    gate, up, down = (torch.zeros(s) for s in shapes)
    for make in (lambda: fp8.Fp8SwigluBlock.from_float(gate, up, down),
                 lambda: fp8.Fp8SwigluBlock.from_blocks(gate, gate, up, up, down, down)):
        with pytest.raises(AhError) as e:
            make()
        assert e.value.status == -1
