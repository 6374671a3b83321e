"""CPU: a workspace's size is planned for the device of the weight, not for the current
one, so a weight whose device cannot be selected has no size.  The handles are made up
here, field by field; sizes read nothing behind their pointers."""
import ctypes as C

import pytest

from agent_harness_b200._lib import lib

ECUDA, EINVAL = -3, -1


class Weight(C.Structure):
    _fields_ = [("tiles", C.c_void_p), ("scales", C.c_void_p), ("rows", C.c_int64), ("cols", C.c_int64),
                ("nt", C.c_int64), ("kb", C.c_int64), ("gate_up", C.c_bool), ("device", C.c_int)]


def weight(rows, cols, gate_up=False, device=63):
    half = rows // 2 if gate_up else rows
    return Weight(0x10000, 0x10000, rows, cols, (half + 127) // 128 * (2 if gate_up else 1), (cols + 127) // 128, gate_up,
                  device)


def test_fields_match_the_library():
    r, c = C.c_int64(), C.c_int64()
    w = weight(300, 1000)
    assert lib().ah_fp8w_shape(C.byref(w), C.byref(r), C.byref(c)) == 0 and (r.value, c.value) == (300, 1000)
    assert lib().ah_fp8w_weight_bytes(C.byref(w)) == 300 * 1000 + 4 * 3 * 8


@pytest.mark.parametrize("m", [1, 40, 65, 260, 2048])
def test_sizes_need_the_weights_device(m):
    n = C.c_size_t(12345)
    w, gu, down = weight(2048, 8192), weight(4096, 512, True), weight(512, 2048)
    assert lib().ah_fp8w_matmul_workspace_bytes(C.byref(w), m, C.byref(n)) == ECUDA
    assert b"device 63" in lib().ah_last_error()
    assert lib().ah_fp8_ffn_workspace_bytes(C.byref(gu), C.byref(down), m, C.byref(n)) == ECUDA
    assert n.value == 12345


def test_a_block_on_two_devices_is_refused():
    n = C.c_size_t()
    gu, down = weight(4096, 512, True, 0), weight(512, 2048, device=1)
    assert lib().ah_fp8_ffn_workspace_bytes(C.byref(gu), C.byref(down), 4, C.byref(n)) == EINVAL
