"""CPU: every refusal of the 8-bit floating point entries comes before the first
CUDA call (fake pointers, no GPU), and the front-end's own checks."""
import ctypes as C

import pytest
import torch

from agent_harness_b200 import fp8
from agent_harness_b200._lib import AhError, lib

P = 0x10000  # stands for an aligned device pointer: never read
OK, EINVAL = 0, -1


def quantize(x=P, ldx=256, dt=0, m=4, k=200, q=P, ldq=208, s=P, lds=2):
    return lib().ah_fp8_quantize(x, ldx, dt, m, k, q, ldq, s, lds, None)


def swiglu(g=P, ldg=256, u=P, ldu=256, dt=1, m=4, k=200, q=P, ldq=208, s=P, lds=2):
    return lib().ah_fp8_swiglu(g, ldg, u, ldu, dt, m, k, q, ldq, s, lds, None)


def norm(x=P, ldx=256, r=P, ldr=256, dt=30, w=P, wdt=1, eps=1e-5, m=4, k=200, q=P, ldq=208, s=P, lds=2):
    return lib().ah_fp8_add_rms_norm(x, ldx, r, ldr, dt, w, wdt, eps, m, k, q, ldq, s, lds, None)


ROW_FAULTS = [dict(m=-1), dict(k=0), dict(dt=2), dict(q=0), dict(q=P + 8), dict(ldq=207), dict(ldq=192), dict(s=0),
              dict(lds=1), dict(m=2**31), dict(k=2**31, ldq=2**31, lds=2**25)]


@pytest.mark.parametrize("entry", [quantize, swiglu, norm])
@pytest.mark.parametrize("fault", ROW_FAULTS)
def test_row_entries_refuse(entry, fault):
    assert entry(**fault) == EINVAL
    assert lib().ah_last_error()


@pytest.mark.parametrize("entry,fault", [
    (quantize, dict(x=0)), (quantize, dict(ldx=199)), (swiglu, dict(g=0)), (swiglu, dict(u=0)),
    (swiglu, dict(ldg=199)), (swiglu, dict(ldu=199)), (norm, dict(x=0)), (norm, dict(w=0)), (norm, dict(wdt=2)),
    (norm, dict(ldx=199)), (norm, dict(ldr=199)), (norm, dict(eps=-1.0)), (norm, dict(eps=float("nan")))])
def test_entry_specific_refusals(entry, fault):
    assert entry(**fault) == EINVAL


@pytest.mark.parametrize("entry,fault", [
    (quantize, dict(x=P + 2)), (quantize, dict(x=P + 1, dt=1)), (quantize, dict(s=P + 2)), (swiglu, dict(g=P + 1)),
    (swiglu, dict(u=P + 3)), (norm, dict(x=P + 1)), (norm, dict(r=P + 1)), (norm, dict(w=P + 1)),
    (norm, dict(w=P + 2, wdt=0))])
def test_pointers_off_their_elements_are_refused(entry, fault):
    assert entry(**fault) == EINVAL
    assert b"aligned to" in lib().ah_last_error()


@pytest.mark.parametrize("entry", [quantize, swiglu, norm])
def test_no_rows_is_a_no_op(entry):
    assert entry(m=0) == OK


def test_weight_makers_refuse():
    h = C.c_void_p()
    L = lib()
    for args in [(0, 200, P, 2, 100, 200), (P, 199, P, 2, 100, 200), (P, 200, 0, 2, 100, 200),
                 (P, 200, P, 1, 100, 200), (P, 200, P, 2, 0, 200), (P, 200, P, 2, 100, 0), (P, 2**31, P, 2**25, 1, 2**30)]:
        assert L.ah_fp8w_from_blocks(*args, C.byref(h), None) == EINVAL
        assert not h.value
    assert L.ah_fp8w_from_blocks(P, 200, P, 2, 100, 200, None, None) == EINVAL
    assert L.ah_fp8w_quantize(P, 200, 2, 100, 200, C.byref(h), None) == EINVAL
    assert L.ah_fp8w_quantize(P, 199, 0, 100, 200, C.byref(h), None) == EINVAL
    assert L.ah_fp8w_from_blocks_gate_up(P, 200, P, 2, 0, 200, P, 2, 100, 200, C.byref(h), None) == EINVAL
    assert L.ah_fp8w_quantize_gate_up(P, 200, P, 199, 0, 100, 200, C.byref(h), None) == EINVAL


def test_weight_makers_refuse_sources_off_their_elements():
    h = C.c_void_p()
    L = lib()
    assert L.ah_fp8w_from_blocks(P, 200, P + 2, 2, 100, 200, C.byref(h), None) == EINVAL
    assert L.ah_fp8w_quantize(P + 2, 200, 0, 100, 200, C.byref(h), None) == EINVAL
    assert L.ah_fp8w_quantize_gate_up(P, 200, P + 1, 200, 1, 100, 200, C.byref(h), None) == EINVAL


def test_null_weights_refused():
    L = lib()
    n, i = C.c_size_t(), C.c_int64()
    assert L.ah_fp8w_matmul(None, P, 208, P, 2, 1, P, 128, 0, None, 0, None) == EINVAL
    assert L.ah_fp8w_matmul_workspace_bytes(None, 1, C.byref(n)) == EINVAL
    assert L.ah_fp8_ffn_workspace_bytes(None, None, 1, C.byref(n)) == EINVAL
    assert L.ah_fp8_ffn(None, None, P, 128, None, 0, 0, P, 1, 1e-5, 1, P, 128, 0, P, 1 << 20, None) == EINVAL
    assert L.ah_fp8w_shape(None, C.byref(i), C.byref(i)) == EINVAL
    assert L.ah_fp8w_weight_bytes(None) == 0
    assert L.ah_fp8w_destroy(None) == OK


def test_front_end_refuses_host_tensors():
    x = torch.zeros(2, 128)
    for fn in (lambda: fp8.quantize_fp8(x), lambda: fp8.swiglu_fp8(x, x),
               lambda: fp8.add_rms_norm_fp8(x, torch.ones(128)), lambda: fp8.Fp8Weight.from_float(x),
               lambda: fp8.Fp8SwigluBlock.from_float(x, x, x.t())):
        with pytest.raises(AhError) as e:
            fn()
        assert e.value.status == EINVAL


def test_alloc_rows_start_at_16_bytes():
    q, s = fp8.alloc(3, 131, "cpu")
    assert q.shape == (3, 131) and q.stride() == (144, 1) and s.shape == (3, 2)
