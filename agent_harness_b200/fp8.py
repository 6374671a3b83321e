"""8-bit floating point projections: activations as e4m3 rows with one f32 scale
per 128 columns, weights as e4m3 with one per 128 x 128 block, and the steps of a
decoder block that run on them (residual add + RMS norm, SwiGLU, products, the
whole feed-forward block).

A quantised matrix is a pair (q, scales): q [m, k] torch.float8_e4m3fn whose rows
start at multiples of 16 bytes (alloc gives such a pair; so does every call here),
scales [m, ceil(k / 128)] f32.  Everything runs on torch's current stream of the
inputs' device, allocates through torch only, and can be captured into a CUDA
graph once a weight has been made.

The products' waits on the device are bounded.  A call whose wait gives up leaves its
outputs unwritten and sets the library's device error word, which no call here reads, since
that would wait for the stream: lib().ah_check_device_error(stream) does, and clears it."""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import AhError, call, check, lib

GROUP = 128
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_E4M3, _F32 = torch.float8_e4m3fn, torch.float32


def _refuse(message: str):
    raise AhError(-1, message)


# The checks below run on every call of a decode step, beside kernels of a few
# microseconds: they read each tensor attribute once, and compare devices by index.

def _rows(t: torch.Tensor, what: str) -> tuple[int, int, int, int]:
    """(rows, columns, row stride, device) of a CUDA matrix with unit-stride columns."""
    shape, dev = t.shape, t.get_device()
    if len(shape) != 2 or dev < 0:
        _refuse(f"{what}: expected a CUDA matrix")
    m, k = shape
    return m, k, k if t.is_contiguous() else _stride(t, m, k, what), dev


def _stride(t: torch.Tensor, m: int, k: int, what: str) -> int:
    ld, unit = t.stride()
    if unit != 1 and k > 1:
        _refuse(f"{what}: expected unit-stride columns")
    if ld < k:
        if m > 1:
            _refuse(f"{what}: rows overlap")
        return k  # a single row's stride is free
    return ld


def _like(t: torch.Tensor, m: int, k: int, device: int, what: str) -> int:
    """The row stride of a second matrix, which has to be [m, k] on that device."""
    if t.shape != (m, k):
        _refuse(f"{what}: expected [{m}, {k}], got {list(t.shape)}")
    if t.get_device() != device:
        _refuse(f"{what}: on another device than the other tensors")
    return k if t.is_contiguous() else _stride(t, m, k, what)


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        _refuse(f"{what}: expected f32, f16 or bf16, got {t.dtype}")
    return code


def _quantised(q: torch.Tensor, scales: torch.Tensor, m: int, k: int, device: int) -> tuple[int, int]:
    """Checks a (q, scales) pair of m rows and k columns: their row strides."""
    if q.dtype is not _E4M3 or scales.dtype is not _F32:
        _refuse("expected q as float8_e4m3fn and scales as float32")
    ldq, lds = _like(q, m, k, device, "q"), _like(scales, m, (k + 127) // 128, device, "scales")
    return (ldq + 15) // 16 * 16 if m <= 1 else ldq, lds  # the stride of one row or none is free


def alloc(m: int, k: int, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """An uninitialised (q, scales) pair for m rows of k columns."""
    q = torch.empty(m, (k + 15) // 16 * 16, dtype=_E4M3, device=device)[:, :k]
    return q, torch.empty(m, (k + GROUP - 1) // GROUP, dtype=torch.float32, device=device)


def _outputs(m: int, k: int, device: int, out, scales):
    if out is None or scales is None:
        if out is not scales:
            _refuse("give out and scales together")
        out, scales = alloc(m, k, torch.device("cuda", device))
    ldq, lds = _quantised(out, scales, m, k, device)
    return out, scales, ldq, lds


_functions: dict = {}
_current_device = torch._C._cuda_getDevice  # what torch.cuda.current_device and current_stream return,
_raw_stream = torch._C._cuda_getCurrentRawStream  # without their wrappers


def _run(device: int, name: str, *args):
    """One library call on the device's current stream."""
    fn = _functions.get(name) or _functions.setdefault(name, getattr(lib(), name))
    if _current_device() == device:
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc:
        check(rc)


def quantize_fp8(x: torch.Tensor, out: torch.Tensor | None = None,
                 scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x [m, k] f32 / f16 / bf16 -> (q, scales)."""
    m, k, ldx, dev = _rows(x, "x")
    dt = _dtype(x, "x")
    out, scales, ldq, lds = _outputs(m, k, dev, out, scales)
    _run(dev, "ah_fp8_quantize", x.data_ptr(), ldx, dt, m, k, out.data_ptr(), ldq, scales.data_ptr(), lds)
    return out, scales


def swiglu_fp8(gate: torch.Tensor, up: torch.Tensor, out: torch.Tensor | None = None,
               scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """silu(gate) * up (inference/ffn.rs:155-174), quantised: gate and up [m, k] of
    one type (halves of one matrix will do) -> (q, scales)."""
    m, k, ldg, dev = _rows(gate, "gate")
    dt, ldu = _dtype(gate, "gate"), _like(up, m, k, dev, "up")
    if up.dtype is not gate.dtype:
        _refuse("gate and up must have one type")
    out, scales, ldq, lds = _outputs(m, k, dev, out, scales)
    _run(dev, "ah_fp8_swiglu", gate.data_ptr(), ldg, up.data_ptr(), ldu, dt, m, k, out.data_ptr(), ldq,
         scales.data_ptr(), lds)
    return out, scales


def _norm_args(x, norm_w, residual):
    m, k, ldx, dev = _rows(x, "x")
    dt, wdt = _dtype(x, "x"), _dtype(norm_w, "norm_w")
    if norm_w.shape != (k,) or norm_w.get_device() != dev or not norm_w.is_contiguous():
        _refuse("norm_w must be one contiguous value per column, on x's device")
    if residual is None:
        return m, k, dev, ldx, dt, wdt, None, 0
    if residual.dtype is not x.dtype:
        _refuse("residual must have x's type")
    return m, k, dev, ldx, dt, wdt, residual.data_ptr(), _like(residual, m, k, dev, "residual")


def add_rms_norm_fp8(x: torch.Tensor, norm_w: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-5,
                     out: torch.Tensor | None = None,
                     scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """residual += x in place (no residual: x alone), then its RMS norm
    (inference/math.rs:53-63) times norm_w [k], quantised -> (q, scales).
    norm_w may be f16 (the decoder's storage), f32 or bf16."""
    m, k, dev, ldx, dt, wdt, rp, ldr = _norm_args(x, norm_w, residual)
    out, scales, ldq, lds = _outputs(m, k, dev, out, scales)
    _run(dev, "ah_fp8_add_rms_norm", x.data_ptr(), ldx, rp, ldr, dt, norm_w.data_ptr(), wdt, eps, m, k,
         out.data_ptr(), ldq, scales.data_ptr(), lds)
    return out, scales


def _blocks_of(q: torch.Tensor, scales: torch.Tensor) -> tuple[int, int]:
    n, k, ldq, dev = _rows(q, "q")
    if q.dtype is not _E4M3 or scales.dtype is not _F32:
        _refuse("expected q as float8_e4m3fn and scales as float32")
    return ldq, _like(scales, (n + GROUP - 1) // GROUP, (k + GROUP - 1) // GROUP, dev, "scales")


class Fp8Weight:
    """A device-resident e4m3 matrix [rows, cols] with a scale per 128 x 128 block."""

    def __init__(self, handle: C.c_void_p, rows: int, cols: int, device: torch.device):
        self._h = handle
        self.rows, self.cols, self.device = rows, cols, device
        self._dev = device.index
        self._bytes = (-1, 0)  # rows and workspace bytes of the last call

    @classmethod
    def _make(cls, name: str, device: torch.device, rows: int, cols: int, *args, n: int | None = None) -> "Fp8Weight":
        h = C.c_void_p()
        with torch.cuda.device(device):
            call(name, *args, rows if n is None else n, cols, C.byref(h), torch.cuda.current_stream().cuda_stream)
        return cls(h, rows, cols, device)

    @classmethod
    def from_blocks(cls, q: torch.Tensor, scales: torch.Tensor) -> "Fp8Weight":
        """q [rows, cols] e4m3, scales [ceil(rows / 128), ceil(cols / 128)] f32 (copied)."""
        ldq, lds = _blocks_of(q, scales)
        return cls._make("ah_fp8w_from_blocks", q.device, *q.shape, q.data_ptr(), ldq, scales.data_ptr(), lds)

    @classmethod
    def from_float(cls, w: torch.Tensor) -> "Fp8Weight":
        """w [rows, cols] f32 / f16 / bf16, quantised on the device."""
        ld, dt = _rows(w, "w")[2], _dtype(w, "w")
        return cls._make("ah_fp8w_quantize", w.device, *w.shape, w.data_ptr(), ld, dt)

    @property
    def handle(self) -> C.c_void_p:
        return self._h

    @property
    def weight_bytes(self) -> int:
        return int(lib().ah_fp8w_weight_bytes(self._h))

    def workspace_bytes(self, m: int) -> int:
        n = C.c_size_t()
        call("ah_fp8w_matmul_workspace_bytes", self._h, m, C.byref(n))
        return int(n.value)

    def matmul(self, q: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None,
               dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """y = dequant(q, scales) @ W^T, [m, rows] in out's type (or dtype), sums in f32."""
        shape, dev = q.shape, self._dev
        m = shape[0] if len(shape) == 2 else -1
        ldq, lds = _quantised(q, scales, m, self.cols, dev)
        if out is None:
            out = torch.empty(m, self.rows, dtype=dtype, device=self.device)
        ldy = _like(out, m, self.rows, dev, "out")
        rows, nbytes = self._bytes
        if rows != m:
            nbytes = self.workspace_bytes(m)
            self._bytes = (m, nbytes)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        _run(dev, "ah_fp8w_matmul", self._h, q.data_ptr(), ldq, scales.data_ptr(), lds, m, out.data_ptr(), ldy,
             _dtype(out, "out"), None if ws is None else ws.data_ptr(), nbytes)
        return out

    def close(self):
        if self._h:
            lib().ah_fp8w_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Fp8SwigluBlock:
    """A decoder's feed-forward block (inference/ffn.rs:72-111 and the norm before
    it, inference/mod.rs:505-545) on e4m3 weights: residual += x, RMS norm, gate and
    up, silu(gate) * up, down."""

    def __init__(self, gate_up: Fp8Weight, down: Fp8Weight):
        self.gate_up, self.down = gate_up, down
        self.n_embd, self.n_ff, self.device = down.rows, down.cols, down.device
        self._dev = down.device.index
        self._bytes = (-1, 0)  # rows and workspace bytes of the last call

    @staticmethod
    def _check(gate, up, down):
        if gate.dim() != 2 or gate.shape != up.shape or down.shape != (gate.shape[1], gate.shape[0]):
            _refuse("expected gate and up [n_ff, n_embd] and down [n_embd, n_ff]")
        if not (gate.device == up.device == down.device and gate.dtype == up.dtype):
            _refuse("gate, up and down must be on one device, gate and up of one type")

    @classmethod
    def from_blocks(cls, gate_q, gate_scales, up_q, up_scales, down_q, down_scales) -> "Fp8SwigluBlock":
        """gate and up [n_ff, n_embd], down [n_embd, n_ff] e4m3, each with its block scales."""
        cls._check(gate_q, up_q, down_q)
        (ldg, lsg), (ldu, lsu) = _blocks_of(gate_q, gate_scales), _blocks_of(up_q, up_scales)
        n_ff, n_embd = gate_q.shape
        down = Fp8Weight.from_blocks(down_q, down_scales)
        gate_up = Fp8Weight._make("ah_fp8w_from_blocks_gate_up", gate_q.device, 2 * n_ff, n_embd, gate_q.data_ptr(), ldg,
                                  gate_scales.data_ptr(), lsg, up_q.data_ptr(), ldu, up_scales.data_ptr(), lsu, n=n_ff)
        return cls(gate_up, down)

    @classmethod
    def from_float(cls, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor) -> "Fp8SwigluBlock":
        """The same from f32 / f16 / bf16 matrices, quantised on the device."""
        cls._check(gate, up, down)
        ldg, ldu, dt = _rows(gate, "gate")[2], _rows(up, "up")[2], _dtype(gate, "gate")
        n_ff, n_embd = gate.shape
        dn = Fp8Weight.from_float(down)
        gate_up = Fp8Weight._make("ah_fp8w_quantize_gate_up", gate.device, 2 * n_ff, n_embd, gate.data_ptr(), ldg,
                                  up.data_ptr(), ldu, dt, n=n_ff)
        return cls(gate_up, dn)

    def workspace_bytes(self, m: int) -> int:
        n = C.c_size_t()
        call("ah_fp8_ffn_workspace_bytes", self.gate_up.handle, self.down.handle, m, C.byref(n))
        return int(n.value)

    def __call__(self, x: torch.Tensor, norm_w: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-5,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """x [m, n_embd] -> the block's output [m, n_embd] in x's type (or out's);
        residual += x in place.  The caller, or the next norm, adds the output to
        the residual."""
        m, k, dev, ldx, dt, wdt, rp, ldr = _norm_args(x, norm_w, residual)
        if k != self.n_embd or dev != self._dev:
            _refuse(f"x must be [m, {self.n_embd}] on {self.device}")
        if out is None:
            out = torch.empty(m, k, dtype=x.dtype, device=self.device)
        ldy = _like(out, m, k, dev, "out")
        rows, nbytes = self._bytes
        if rows != m:
            nbytes = self.workspace_bytes(m)
            self._bytes = (m, nbytes)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        _run(dev, "ah_fp8_ffn", self.gate_up.handle, self.down.handle, x.data_ptr(), ldx, rp, ldr, dt,
             norm_w.data_ptr(), wdt, eps, m, out.data_ptr(), ldy, _dtype(out, "out"), ws.data_ptr(), nbytes)
        return out

    def close(self):
        self.gate_up.close()
        self.down.close()
