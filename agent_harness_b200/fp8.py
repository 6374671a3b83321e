"""8-bit floating point projections: activations as e4m3 rows with one f32 scale
per 128 columns, weights as e4m3 with one per 128 x 128 block, and the steps of a
decoder block that run on them (residual add + RMS norm, SwiGLU, products, the
whole feed-forward block).

A quantised matrix is a pair (q, scales): q [m, k] torch.float8_e4m3fn whose rows
start at multiples of 16 bytes (alloc gives such a pair; so does every call here),
scales [m, ceil(k / 128)] f32.  Everything runs on torch's current stream of the
inputs' device, allocates through torch only, and can be captured into a CUDA
graph once a weight has been made."""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import AhError, call, lib

GROUP = 128
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_E4M3 = torch.float8_e4m3fn


def _refuse(message: str):
    raise AhError(-1, message)


def _rows(t: torch.Tensor, what: str, like: torch.Tensor | None = None) -> int:
    """The row stride of a CUDA matrix with unit-stride columns."""
    if t.dim() != 2 or not t.is_cuda:
        _refuse(f"{what}: expected a CUDA matrix")
    if like is not None and t.device != like.device:
        _refuse(f"{what}: on another device than the other tensors")
    m, k = t.shape
    if k > 1 and t.stride(1) != 1:
        _refuse(f"{what}: expected unit-stride columns")
    ld = t.stride(0) if m > 1 else max(k, t.stride(0))
    if ld < k:
        _refuse(f"{what}: rows overlap")
    return ld


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        _refuse(f"{what}: expected f32, f16 or bf16, got {t.dtype}")
    return code


def _quantised(q: torch.Tensor, scales: torch.Tensor, like: torch.Tensor | None = None) -> tuple[int, int]:
    """Checks a (q, scales) pair; returns its row strides."""
    ldq, lds = _rows(q, "q", like), _rows(scales, "scales", q)
    if q.dtype != _E4M3 or scales.dtype != torch.float32:
        _refuse("expected q as float8_e4m3fn and scales as float32")
    m, k = q.shape
    if scales.shape[0] != m or scales.shape[1] != (k + GROUP - 1) // GROUP:
        _refuse("scales must be [rows, ceil(columns / 128)]")
    if m <= 1:  # a single row's stride is free
        ldq = (ldq + 15) // 16 * 16
    return ldq, lds


def alloc(m: int, k: int, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """An uninitialised (q, scales) pair for m rows of k columns."""
    q = torch.empty(m, (k + 15) // 16 * 16, dtype=_E4M3, device=device)[:, :k]
    return q, torch.empty(m, (k + GROUP - 1) // GROUP, dtype=torch.float32, device=device)


def _outputs(x: torch.Tensor, out, scales) -> tuple[torch.Tensor, torch.Tensor, int, int]:
    m, k = x.shape
    if (out is None) != (scales is None):
        _refuse("give out and scales together")
    if out is None:
        out, scales = alloc(m, k, x.device)
    elif out.shape != x.shape:
        _refuse("out must have the input's shape")
    ldq, lds = _quantised(out, scales, x)
    return out, scales, ldq, lds


def _run(device: torch.device, name: str, *args):
    """One library call on the device's current stream."""
    if device.index == torch.cuda.current_device():
        call(name, *args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            call(name, *args, torch.cuda.current_stream(device).cuda_stream)


def quantize_fp8(x: torch.Tensor, out: torch.Tensor | None = None,
                 scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x [m, k] f32 / f16 / bf16 -> (q, scales)."""
    ldx, dt = _rows(x, "x"), _dtype(x, "x")
    out, scales, ldq, lds = _outputs(x, out, scales)
    m, k = x.shape
    _run(x.device, "ah_fp8_quantize", x.data_ptr(), ldx, dt, m, k, out.data_ptr(), ldq, scales.data_ptr(), lds)
    return out, scales


def swiglu_fp8(gate: torch.Tensor, up: torch.Tensor, out: torch.Tensor | None = None,
               scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """silu(gate) * up (inference/ffn.rs:155-174), quantised: gate and up [m, k] of
    one type (halves of one matrix will do) -> (q, scales)."""
    ldg, ldu, dt = _rows(gate, "gate"), _rows(up, "up", gate), _dtype(gate, "gate")
    if up.shape != gate.shape or up.dtype != gate.dtype:
        _refuse("gate and up must have one shape and type")
    out, scales, ldq, lds = _outputs(gate, out, scales)
    m, k = gate.shape
    _run(gate.device, "ah_fp8_swiglu", gate.data_ptr(), ldg, up.data_ptr(), ldu, dt, m, k, out.data_ptr(), ldq,
         scales.data_ptr(), lds)
    return out, scales


def _norm_args(x, norm_w, residual):
    ldx, dt = _rows(x, "x"), _dtype(x, "x")
    wdt = _dtype(norm_w, "norm_w")
    if norm_w.shape != (x.shape[1],) or not norm_w.is_contiguous() or norm_w.device != x.device:
        _refuse("norm_w must be one contiguous value per column, on x's device")
    rp, ldr = None, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            _refuse("residual must have x's shape and type")
        rp, ldr = residual.data_ptr(), _rows(residual, "residual", x)
    return ldx, dt, wdt, rp, ldr


def add_rms_norm_fp8(x: torch.Tensor, norm_w: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-5,
                     out: torch.Tensor | None = None,
                     scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """residual += x in place (no residual: x alone), then its RMS norm
    (inference/math.rs:53-63) times norm_w [k], quantised -> (q, scales).
    norm_w may be f16 (the decoder's storage), f32 or bf16."""
    ldx, dt, wdt, rp, ldr = _norm_args(x, norm_w, residual)
    out, scales, ldq, lds = _outputs(x, out, scales)
    m, k = x.shape
    _run(x.device, "ah_fp8_add_rms_norm", x.data_ptr(), ldx, rp, ldr, dt, norm_w.data_ptr(), wdt, eps, m, k,
         out.data_ptr(), ldq, scales.data_ptr(), lds)
    return out, scales


def _blocks_of(q: torch.Tensor, scales: torch.Tensor) -> tuple[int, int]:
    ldq, lds = _rows(q, "q"), _rows(scales, "scales", q)
    if q.dtype != _E4M3 or scales.dtype != torch.float32:
        _refuse("expected q as float8_e4m3fn and scales as float32")
    if scales.shape != tuple((n + GROUP - 1) // GROUP for n in q.shape):
        _refuse("scales must be [ceil(rows / 128), ceil(columns / 128)]")
    return ldq, lds


class Fp8Weight:
    """A device-resident e4m3 matrix [rows, cols] with a scale per 128 x 128 block."""

    def __init__(self, handle: C.c_void_p, rows: int, cols: int, device: torch.device):
        self._h = handle
        self.rows, self.cols, self.device = rows, cols, device

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
        ld, dt = _rows(w, "w"), _dtype(w, "w")
        return cls._make("ah_fp8w_quantize", w.device, *w.shape, w.data_ptr(), ld, dt)

    @property
    def handle(self) -> C.c_void_p:
        return self._h

    @property
    def weight_bytes(self) -> int:
        return int(lib().ah_fp8w_weight_bytes(self._h))

    def matmul(self, q: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None,
               dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """y = dequant(q, scales) @ W^T, [m, rows] in out's type (or dtype), sums in f32."""
        ldq, lds = _quantised(q, scales)
        if q.shape[1] != self.cols or q.device != self.device:
            _refuse(f"q must be [m, {self.cols}] on {self.device}")
        m = q.shape[0]
        if out is None:
            out = torch.empty(m, self.rows, dtype=dtype, device=q.device)
        elif out.shape != (m, self.rows):
            _refuse(f"out must be [{m}, {self.rows}]")
        ldy, dt = _rows(out, "out", q), _dtype(out, "out")
        _run(self.device, "ah_fp8w_matmul", self._h, q.data_ptr(), ldq, scales.data_ptr(), lds, m, out.data_ptr(), ldy,
             dt)
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

    @staticmethod
    def _check(gate, up, down):
        if gate.shape != up.shape or down.shape != (gate.shape[1], gate.shape[0]):
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
        ldg, ldu, dt = _rows(gate, "gate"), _rows(up, "up"), _dtype(gate, "gate")
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
        ldx, dt, wdt, rp, ldr = _norm_args(x, norm_w, residual)
        if x.shape[1] != self.n_embd or x.device != self.device:
            _refuse(f"x must be [m, {self.n_embd}] on {self.device}")
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        elif out.shape != x.shape:
            _refuse("out must have x's shape")
        ldy, odt = _rows(out, "out", x), _dtype(out, "out")
        m = x.shape[0]
        ws = torch.empty(self.workspace_bytes(m), dtype=torch.uint8, device=x.device)
        _run(self.device, "ah_fp8_ffn", self.gate_up.handle, self.down.handle, x.data_ptr(), ldx, rp, ldr, dt,
             norm_w.data_ptr(), wdt, eps, m, out.data_ptr(), ldy, odt, ws.data_ptr(), ws.numel())
        return out

    def close(self):
        self.gate_up.close()
        self.down.close()
