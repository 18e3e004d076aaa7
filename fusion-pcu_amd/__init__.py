"""fusion_pcu_amd — MI355X-native (gfx950) strict owned-tensor backend for Fusion PCU.

The product is ``libpcu_rocm.so`` (hand-written HIP kernels + C ABI, include/pcu_rocm.h).
This package is the host-side mirror of the reference facade for the strict path: the
error/fault vocabulary (``PcuExecutionError``, ``PcuExecutionFault``), device-resident
tensors, the op-level calls, programs with one terminal synchronization, and the graph
capture API (``pcu.matmul``, ``pcu.relu``, ``pcu.mean_squared_error``, ``pcu.gradient(s)``,
``pcu.sgd_update``) in ``fusion_pcu_amd.graph``. Every arithmetic call runs on the GPU
through the C ABI; there is no CPU fallback.
"""
from __future__ import annotations

import contextlib
import ctypes
import enum
import operator
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import numpy as np

from . import _abi

__all__ = [
    "PcuExecutionFaultKind", "TensorArithmeticStep", "PcuFloatUnderflowPolicy",
    "PcuExecutionFault", "CompoundFault", "PcuExecutionError", "Context", "DeviceArray",
    "lib", "library_path", "bfloat16", "to_bfloat16", "from_bfloat16",
]


def lib():
    return _abi.load()


def library_path() -> str:
    return _abi.LIB_PATH


class PcuExecutionFaultKind(enum.IntEnum):
    """core/core.rs:25-41 (numbered as the packed fault word)."""
    DivideByZero = 1
    SignedDivisionOverflow = 2
    ArithmeticOverflow = 3
    ArithmeticUnderflow = 4
    InvalidFloatingOperand = 5


class TensorArithmeticStep(enum.IntEnum):
    """core/dialect/tensor.rs:425-430; NONE marks an elementwise ArithmeticFault."""
    NONE = 0
    Multiply = 1
    Add = 2
    Subtract = 3
    Divide = 4


class PcuFloatUnderflowPolicy(enum.IntEnum):
    """core/scalar_float_underflow.rs:47-58."""
    IeeeAfterRounding = 0
    RejectSubnormalResult = 1
    AllowGradualUnderflow = 2


@dataclass(frozen=True)
class PcuExecutionFault:
    """core/core.rs:50-66: kind + the row-major output element as invocation id."""
    kind: PcuExecutionFaultKind
    invocation_id: int
    recovered: bool = False


@dataclass(frozen=True)
class CompoundFault:
    """TensorError::{ArithmeticFault, CompoundArithmeticFault} (core/dialect/tensor.rs:
    234-252): the faulting node, output element, reduction index and step."""
    node: int
    element_index: int
    reduction_index: int
    step: TensorArithmeticStep
    kind: PcuExecutionFaultKind

    @property
    def compound(self) -> bool:
        return self.step != TensorArithmeticStep.NONE


class PcuExecutionError(Exception):
    """fusion-pcu/global.rs:195-275. ``status`` is the C ABI status; an arithmetic fault
    carries ``tensor_fault`` (the structured TensorError coordinates)."""

    def __init__(self, status: int, message: str, tensor_fault: Optional[CompoundFault] = None):
        self.status = status
        self.message = message
        self.tensor_fault = tensor_fault
        super().__init__(f"{_abi.STATUS_NAMES.get(status, status)}: {message}")

    def arithmetic_fault(self) -> Optional[PcuExecutionFault]:
        """fusion-pcu/global.rs:392-449: the element index as invocation id."""
        if self.tensor_fault is None:
            return None
        return PcuExecutionFault(self.tensor_fault.kind, self.tensor_fault.element_index, False)


_NP_DTYPE = {np.dtype(np.float32): _abi.PCU_F32, np.dtype(np.float64): _abi.PCU_F64}


def dtype_code(dtype) -> int:
    try:
        return _NP_DTYPE[np.dtype(dtype)]
    except KeyError:
        raise PcuExecutionError(_abi.PCU_ERR_UNSUPPORTED, f"unsupported scalar type {dtype}")


# numpy has no bfloat16: arrays of this type hold the upper halves of binary32 bit patterns.
bfloat16 = np.dtype([("bfloat16", np.uint16)])


def to_bfloat16(x) -> np.ndarray:
    """binary32 values rounded to nearest even (a NaN stays a NaN)."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    b = x.view(np.uint32)
    r = ((b.astype(np.uint64) + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    r = np.where(np.isnan(x), ((b >> 16) | 0x40).astype(np.uint16), r)
    return np.ascontiguousarray(r).view(bfloat16).reshape(x.shape)


def from_bfloat16(x: np.ndarray) -> np.ndarray:
    return (np.ascontiguousarray(x).view(np.uint16).astype(np.uint32) << 16).view(np.float32).reshape(x.shape)


_LOGIT_DTYPE = {np.dtype(np.float32): _abi.PCU_F32, np.dtype(np.float64): _abi.PCU_F64,
                bfloat16: _abi.PCU_BF16, np.dtype(np.float16): _abi.PCU_F16}


def _logit_code(what: str, dtype) -> int:
    try:
        return _LOGIT_DTYPE[dtype]
    except KeyError:
        raise PcuExecutionError(_abi.PCU_ERR_UNSUPPORTED, f"{what}: unsupported scalar type {dtype}")


_FLOAT32, _FLOAT64, _INT32 = np.dtype(np.float32), np.dtype(np.float64), np.dtype(np.int32)


def _stat_dtype(dtype) -> np.dtype:
    """The type of a row's statistics: binary32, binary64 for binary64 rows."""
    return _FLOAT64 if dtype is _FLOAT64 or dtype == _FLOAT64 else _FLOAT32


def _need(what: str, x: "DeviceArray", shape: Tuple[int, ...], dtype: np.dtype) -> None:
    """_require on a path that a token takes: shape a tuple, dtype a numpy dtype."""
    if x.shape != shape or (x.dtype is not dtype and x.dtype != dtype):
        _require(what, x, shape, dtype)


def _require(what: str, x: "DeviceArray", shape, dtype) -> None:
    """TensorError::ShapeMismatch / ScalarTypeMismatch before any pointer reaches the C ABI:
    the kernels take one element count and raw pointers, so a smaller or narrower buffer
    would be read or written past its end."""
    if x.shape != tuple(shape) or x.dtype != np.dtype(dtype):
        raise PcuExecutionError(
            _abi.PCU_ERR_SHAPE,
            f"ShapeMismatch: {what} is {x.shape} {x.dtype}, expected {tuple(shape)} {np.dtype(dtype)}")


def _fault_from(f: _abi.Fault) -> CompoundFault:
    return CompoundFault(int(f.node), int(f.element_index), int(f.reduction_index),
                         TensorArithmeticStep(int(f.step)), PcuExecutionFaultKind(int(f.kind)))


class DeviceArray:
    """A dense row-major device allocation owned by a Context (the resident backing of a
    PcuTensor; fusion-pcu/global/arguments.rs:636-690)."""

    def __init__(self, ctx: "Context", ptr: int, shape: Tuple[int, ...], dtype):
        self.ctx = ctx
        self.ptr = ptr
        self.shape = tuple(int(s) for s in shape)
        self.dtype = np.dtype(dtype)

    @classmethod
    def _of(cls, ctx: "Context", ptr: int, shape: Tuple[int, ...], dtype: np.dtype) -> "DeviceArray":
        """Wrap a pointer whose shape (a tuple of ints) and dtype (a numpy dtype) are already
        normalized: the per-call path of prepared programs."""
        a = cls.__new__(cls)
        a.ctx = ctx
        a.ptr = ptr
        a.shape = shape
        a.dtype = dtype
        return a

    @property
    def size(self) -> int:
        return int(np.prod(self.shape, dtype=np.int64)) if self.shape else 1

    @property
    def nbytes(self) -> int:
        return self.size * self.dtype.itemsize

    def numpy(self) -> np.ndarray:
        out = np.empty(self.shape, dtype=self.dtype)
        self.ctx.download_into(out, self)
        return out

    def free(self) -> None:
        if self.ptr:
            self.ctx.free(self)

    def __repr__(self) -> str:
        return f"DeviceArray(shape={self.shape}, dtype={self.dtype}, ptr=0x{self.ptr:x})"


class Context:
    """One pcu_ctx: a device, its ordered stream, memory pool and fault records."""

    def __init__(self, device: int = 0):
        self._lib = lib()
        handle = ctypes.c_void_p()
        st = self._lib.pcu_ctx_open(device, ctypes.byref(handle))
        if st != _abi.PCU_OK:
            raise PcuExecutionError(st, self._lib.pcu_last_error(None).decode())
        self.handle = handle
        self.device = device
        self._program_nodes = None

    # ---------------------------------------------------------------- basics
    def close(self) -> None:
        if self.handle:
            self._lib.pcu_ctx_close(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def error_text(self) -> str:
        return self._lib.pcu_last_error(self.handle).decode()

    def check(self, st: int, fault: Optional[_abi.Fault] = None) -> None:
        if st == _abi.PCU_OK:
            return
        if st == _abi.PCU_ARITHMETIC_FAULT and fault is not None:
            tf = _fault_from(fault)
            raise PcuExecutionError(st, f"arithmetic fault {tf}", tf)
        raise PcuExecutionError(st, self.error_text())

    def synchronize(self) -> None:
        self.check(self._lib.pcu_ctx_synchronize(self.handle))

    MATMUL_ENGINES = {"auto": 0, "valu": 1, "mfma_products": 2}

    def last_fault(self) -> Optional[CompoundFault]:
        """First fault of the most recent program or op call (pcu_fault_read), or None."""
        f = _abi.Fault()
        st = self._lib.pcu_fault_read(self.handle, ctypes.byref(f))
        if st == _abi.PCU_OK:
            return None
        if st != _abi.PCU_ARITHMETIC_FAULT:
            self.check(st)
        return _fault_from(f)

    def reset_fault(self) -> None:
        """Forget the held fault (pcu_fault_reset)."""
        self.check(self._lib.pcu_fault_reset(self.handle))

    def set_matmul_engine(self, engine: str) -> None:
        """Engine of the strict MatMul ("auto", "valu", "mfma_products"); every engine gives
        the same bits and first fault. "auto" runs products of few cells, where one launch is
        the faster way, as one launch on the vector unit and the other F32 ones with
        matrix-core products; "valu" and "mfma_products" always take the screened tile
        kernels."""
        self.check(self._lib.pcu_ctx_set_matmul_engine(self.handle, self.MATMUL_ENGINES[engine]))

    @property
    def stream(self) -> int:
        return self._lib.pcu_ctx_stream(self.handle)

    # ---------------------------------------------------------------- memory
    def empty(self, shape: Sequence[int], dtype) -> DeviceArray:
        shape = tuple(int(s) for s in shape)
        n = int(np.prod(shape, dtype=np.int64)) if shape else 1
        p = ctypes.c_void_p()
        self.check(self._lib.pcu_buf_alloc(self.handle, n * np.dtype(dtype).itemsize, ctypes.byref(p)))
        return DeviceArray(self, p.value, shape, dtype)

    def upload(self, host: np.ndarray) -> DeviceArray:
        host = np.ascontiguousarray(host)
        dev = self.empty(host.shape, host.dtype)
        self.upload_into(dev, host)
        return dev

    def upload_into(self, dev: DeviceArray, host: np.ndarray) -> None:
        host = np.ascontiguousarray(host, dtype=dev.dtype)
        if host.nbytes != dev.nbytes:
            raise PcuExecutionError(_abi.PCU_ERR_ARGUMENT, "upload size mismatch")
        self.check(self._lib.pcu_upload(self.handle, dev.ptr, host.ctypes.data, host.nbytes))

    def download_into(self, host: np.ndarray, dev: DeviceArray) -> None:
        if not host.flags.c_contiguous or host.nbytes != dev.nbytes:
            raise PcuExecutionError(_abi.PCU_ERR_ARGUMENT, "download size mismatch")
        self.check(self._lib.pcu_download(self.handle, host.ctypes.data, dev.ptr, dev.nbytes))

    def free(self, dev: DeviceArray) -> None:
        self.check(self._lib.pcu_buf_free(self.handle, dev.ptr))
        dev.ptr = 0

    # --------------------------------------------------------------- program
    @contextlib.contextmanager
    def program(self):
        """Enqueue several ops and synchronize once; raises PcuExecutionError carrying
        the first fault in node order."""
        self.check(self._lib.pcu_program_begin(self.handle))
        ok = False
        try:
            yield self
            ok = True
        finally:
            f = _abi.Fault()
            st = self._lib.pcu_program_end(self.handle, ctypes.byref(f))
            if ok:
                self.check(st, f)

    def next_node(self) -> int:
        return int(self._lib.pcu_program_next_node(self.handle))

    def mark(self, slot: int) -> None:
        self.check(self._lib.pcu_mark(self.handle, slot))

    def elapsed_ms(self, a: int, b: int) -> float:
        ms = ctypes.c_float()
        self.check(self._lib.pcu_elapsed_ms(self.handle, a, b, ctypes.byref(ms)))
        return float(ms.value)

    def profile(self, on: bool = True) -> None:
        """Start (and reset) or stop per-kernel HIP-event timing."""
        self.check(self._lib.pcu_profile_enable(self.handle, int(on)))

    def kernel_time(self, kernel: str) -> Tuple[float, int]:
        """(total milliseconds, launches) of one kernel since profile(True)."""
        ms = ctypes.c_double()
        n = ctypes.c_uint64()
        self.check(self._lib.pcu_profile_read(self.handle, _abi.KERNEL_IDS[kernel],
                                              ctypes.byref(ms), ctypes.byref(n)))
        return float(ms.value), int(n.value)

    def calibrate_direct_copy(self, src: "DeviceArray", dst: "DeviceArray") -> None:
        """Measurement aid: copy src into dst (same byte size, a multiple of 4 KiB) reading
        with the direct global-to-LDS load of the matrix-core MatMul tiles (see
        pcu_calibrate_direct_copy); synchronizes."""
        if src.nbytes != dst.nbytes:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, "calibration copy: sizes differ")
        self.check(self._lib.pcu_calibrate_direct_copy(self.handle, src.ptr, dst.ptr, src.nbytes))

    # ------------------------------------------------------------------- ops
    def _call(self, fn, *args) -> None:
        f = _abi.Fault()
        st = fn(self.handle, *args, ctypes.byref(f))
        self.check(st, f)

    def strict_matmul(self, a: DeviceArray, b: DeviceArray, transpose_left=False,
                      transpose_right=False, policy=0, out: Optional[DeviceArray] = None):
        if len(a.shape) != 2 or len(b.shape) != 2 or a.dtype != b.dtype:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"MatMulShape {a.shape} x {b.shape}")
        rows, inner = (a.shape[1], a.shape[0]) if transpose_left else a.shape
        inner_b, cols = (b.shape[1], b.shape[0]) if transpose_right else b.shape
        if inner != inner_b:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"MatMulShape {a.shape} x {b.shape}")
        if out is None:
            out = self.empty((rows, cols), a.dtype)
        _require("out", out, (rows, cols), a.dtype)
        self._call(self._lib.pcu_strict_matmul, dtype_code(a.dtype), rows, inner, cols,
                   int(transpose_left), int(transpose_right), a.ptr, b.ptr, out.ptr, int(policy))
        return out

    def checked_binary(self, op: int, a: DeviceArray, b, policy=0, out=None):
        if isinstance(b, DeviceArray):
            _require("right", b, a.shape, a.dtype)
        if out is None:
            out = self.empty(a.shape, a.dtype)
        _require("out", out, a.shape, a.dtype)
        if isinstance(b, DeviceArray):
            self._call(self._lib.pcu_checked_binary, dtype_code(a.dtype), op, a.size, a.ptr,
                       b.ptr, out.ptr, int(policy))
        else:
            bits = int(np.array(b, dtype=a.dtype).view(np.uint32 if a.dtype == np.float32 else np.uint64))
            self._call(self._lib.pcu_checked_binary_uniform, dtype_code(a.dtype), op, a.size,
                       a.ptr, bits, out.ptr, int(policy))
        return out

    def checked_relu(self, x: DeviceArray, policy=0, out=None):
        if out is None:
            out = self.empty(x.shape, x.dtype)
        _require("out", out, x.shape, x.dtype)
        self._call(self._lib.pcu_checked_relu, dtype_code(x.dtype), x.size, x.ptr, out.ptr, int(policy))
        return out

    def checked_relu_backward(self, x: DeviceArray, up: DeviceArray, policy=0, out=None):
        _require("upstream", up, x.shape, x.dtype)
        if out is None:
            out = self.empty(x.shape, x.dtype)
        _require("out", out, x.shape, x.dtype)
        self._call(self._lib.pcu_checked_relu_backward, dtype_code(x.dtype), x.size, x.ptr,
                   up.ptr, out.ptr, int(policy))
        return out

    def checked_add_relu(self, a: DeviceArray, b: DeviceArray, policy=0, out=None):
        _require("right", b, a.shape, a.dtype)
        if out is None:
            out = self.empty(a.shape, a.dtype)
        _require("out", out, a.shape, a.dtype)
        self._call(self._lib.pcu_checked_add_relu, dtype_code(a.dtype), a.size, a.ptr, b.ptr,
                   out.ptr, int(policy))
        return out

    def strict_sgd(self, w: DeviceArray, g: DeviceArray, learning_rate: float, policy=0, out=None):
        _require("gradient", g, w.shape, w.dtype)
        if out is None:
            out = self.empty(w.shape, w.dtype)
        _require("out", out, w.shape, w.dtype)
        self._call(self._lib.pcu_strict_sgd, dtype_code(w.dtype), w.size, w.ptr, g.ptr,
                   float(np.float32(learning_rate)), out.ptr, int(policy))
        return out

    def strict_mse(self, p: DeviceArray, t: DeviceArray, policy=0, out=None):
        _require("target", t, p.shape, p.dtype)
        if out is None:
            out = self.empty((), p.dtype)
        _require("out", out, (), p.dtype)
        self._call(self._lib.pcu_strict_mse, dtype_code(p.dtype), p.size, p.ptr, t.ptr,
                   out.ptr, int(policy))
        return out

    # ------------------------------------------------ native compound arithmetic
    # Explicitly permitted native compounds (Boundary + BackendDefined): backend-defined
    # order, contraction and special values; no arithmetic fault is raised.
    def native_matmul(self, a: DeviceArray, b: DeviceArray, transpose_left=False,
                      transpose_right=False, out: Optional[DeviceArray] = None):
        if len(a.shape) != 2 or len(b.shape) != 2 or a.dtype != b.dtype:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"MatMulShape {a.shape} x {b.shape}")
        rows, inner = (a.shape[1], a.shape[0]) if transpose_left else a.shape
        inner_b, cols = (b.shape[1], b.shape[0]) if transpose_right else b.shape
        if inner != inner_b:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"MatMulShape {a.shape} x {b.shape}")
        if out is None:
            out = self.empty((rows, cols), a.dtype)
        _require("out", out, (rows, cols), a.dtype)
        self.check(self._lib.pcu_native_matmul(self.handle, dtype_code(a.dtype), rows, inner, cols,
                                               int(transpose_left), int(transpose_right), a.ptr,
                                               b.ptr, out.ptr))
        return out

    def native_mse(self, p: DeviceArray, t: DeviceArray, out=None):
        _require("target", t, p.shape, p.dtype)
        if out is None:
            out = self.empty((), p.dtype)
        _require("out", out, (), p.dtype)
        self.check(self._lib.pcu_native_mse(self.handle, dtype_code(p.dtype), p.size, p.ptr, t.ptr,
                                            out.ptr))
        return out

    def native_sgd(self, w: DeviceArray, g: DeviceArray, learning_rate: float, contracted=False,
                   out=None):
        _require("gradient", g, w.shape, w.dtype)
        if out is None:
            out = self.empty(w.shape, w.dtype)
        _require("out", out, w.shape, w.dtype)
        self.check(self._lib.pcu_native_sgd(self.handle, dtype_code(w.dtype), w.size, w.ptr, g.ptr,
                                            float(np.float32(learning_rate)), int(contracted),
                                            out.ptr))
        return out

    # ------------------------------------------------------ operators on logits
    # Logits are a [rows, columns] array of float32, float64, float16 or ``bfloat16``; ``vocab``
    # (default: all columns) names how many leading columns are real where the rest is
    # padding. Results that are not passed in are allocated.
    def _logits(self, what: str, x: DeviceArray, vocab: Optional[int]) -> _abi.Logits:
        code = _logit_code(what, x.dtype)
        if len(x.shape) != 2 or (vocab is not None and not 0 <= vocab <= x.shape[1]):
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"{what}: {x.shape} with vocab {vocab}")
        return _abi.Logits(x.ptr, code, 0, x.shape[0], x.shape[1] if vocab is None else vocab, x.shape[1])

    def _out(self, what: str, x: Optional[DeviceArray], shape, dtype) -> DeviceArray:
        if x is None:
            return self.empty(shape, dtype)
        _need(what, x, shape, dtype)
        return x

    def native_top_logits(self, logits: DeviceArray, k: int, temperature: float = 1.0,
                          vocab: Optional[int] = None, values: Optional[DeviceArray] = None,
                          indices: Optional[DeviceArray] = None,
                          log_sum: Optional[DeviceArray] = None):
        """The k largest logits of each row by (value descending, index ascending), their int32
        indices, and the row's log(sum exp(l / temperature)): ``(values, indices, log_sum)``,
        a teacher's side of the distillation below (pcu_native_top_logits)."""
        lg = self._logits("top_logits", logits, vocab)
        k = int(k)
        if not 0 <= k <= _abi.LOGITS_MAX_K:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"top_logits: k {k} is not in [0, {_abi.LOGITS_MAX_K}]")
        rows = logits.shape[0]
        values = self._out("values", values, (rows, k), logits.dtype)
        indices = self._out("indices", indices, (rows, k), _INT32)
        log_sum = self._out("log_sum", log_sum, (rows,), _stat_dtype(logits.dtype))
        self.check(self._lib.pcu_native_top_logits(self.handle, ctypes.byref(lg), k, temperature, values.ptr,
                                                   indices.ptr, log_sum.ptr))
        return values, indices, log_sum

    def _distill(self, student: DeviceArray, teacher_values: DeviceArray, teacher_indices: DeviceArray,
                 teacher_log_sum, labels, temperature: float, distill_weight: float, label_weight: float,
                 vocab: Optional[int]):
        lg = self._logits("distill", student, vocab)
        rows = student.shape[0]
        if len(teacher_values.shape) != 2:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"distill: teacher values are {teacher_values.shape}")
        k = teacher_values.shape[1]
        if k > _abi.LOGITS_MAX_K:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"distill: {k} entries a row are beyond {_abi.LOGITS_MAX_K}")
        code = _logit_code("teacher values", teacher_values.dtype)
        _need("teacher values", teacher_values, (rows, k), teacher_values.dtype)
        _need("teacher indices", teacher_indices, (rows, k), _INT32)
        if teacher_log_sum is not None:
            _need("teacher log-sum", teacher_log_sum, (rows,), _stat_dtype(teacher_values.dtype))
        if labels is not None:
            _need("labels", labels, (rows,), _INT32)
        return lg, _abi.Distill(teacher_values.ptr, teacher_indices.ptr,
                                teacher_log_sum.ptr if teacher_log_sum is not None else None,
                                labels.ptr if labels is not None else None, code, k, temperature,
                                distill_weight, label_weight)

    def native_distill_loss(self, student: DeviceArray, teacher_values: DeviceArray,
                            teacher_indices: DeviceArray, teacher_log_sum: Optional[DeviceArray] = None,
                            labels: Optional[DeviceArray] = None, temperature: float = 1.0,
                            distill_weight: float = 1.0, label_weight: float = 0.0,
                            vocab: Optional[int] = None, loss: Optional[DeviceArray] = None,
                            log_sums: Optional[DeviceArray] = None):
        """Each row's distillation loss against a teacher's top logits (entries with a negative
        index are absent), plus ``label_weight`` times the cross entropy of its label (negative:
        none); without ``teacher_log_sum`` the teacher's probabilities are normalised over the
        row's entries. Returns ``(loss [rows], log_sums [rows, 2])``; see pcu_distill for the
        formulas."""
        lg, d = self._distill(student, teacher_values, teacher_indices, teacher_log_sum, labels, temperature,
                              distill_weight, label_weight, vocab)
        rows, stat = student.shape[0], _stat_dtype(student.dtype)
        loss = self._out("loss", loss, (rows,), stat)
        log_sums = self._out("log_sums", log_sums, (rows, 2), stat)
        self._call(self._lib.pcu_native_distill_loss, ctypes.byref(lg), ctypes.byref(d), loss.ptr, log_sums.ptr)
        return loss, log_sums

    def native_distill_backward(self, student: DeviceArray, teacher_values: DeviceArray,
                                teacher_indices: DeviceArray, log_sums: DeviceArray,
                                teacher_log_sum: Optional[DeviceArray] = None,
                                labels: Optional[DeviceArray] = None, temperature: float = 1.0,
                                distill_weight: float = 1.0, label_weight: float = 0.0,
                                vocab: Optional[int] = None, row_scale: Optional[DeviceArray] = None,
                                gradient: Optional[DeviceArray] = None) -> DeviceArray:
        """The loss's gradient by the student's logits, each row times its ``row_scale``, from
        native_distill_loss's ``log_sums``: an array like ``student`` (padding columns are 0),
        which may be ``student`` itself."""
        lg, d = self._distill(student, teacher_values, teacher_indices, teacher_log_sum, labels, temperature,
                              distill_weight, label_weight, vocab)
        (rows, cols), stat = student.shape, _stat_dtype(student.dtype)
        _need("log_sums", log_sums, (rows, 2), stat)
        if row_scale is not None:
            _need("row_scale", row_scale, (rows,), stat)
        gradient = self._out("gradient", gradient, student.shape, student.dtype)
        self._call(self._lib.pcu_native_distill_backward, ctypes.byref(lg), ctypes.byref(d), log_sums.ptr,
                   row_scale.ptr if row_scale is not None else None, gradient.ptr, cols, cols)
        return gradient

    def native_distill_step(self, student: DeviceArray, teacher_values: DeviceArray,
                            teacher_indices: DeviceArray, teacher_log_sum: Optional[DeviceArray] = None,
                            labels: Optional[DeviceArray] = None, temperature: float = 1.0,
                            distill_weight: float = 1.0, label_weight: float = 0.0,
                            vocab: Optional[int] = None, row_scale: Optional[DeviceArray] = None,
                            loss: Optional[DeviceArray] = None, gradient: Optional[DeviceArray] = None):
        """native_distill_loss and native_distill_backward in one call, which reads the logits once
        where it can: ``(loss [rows], gradient)``."""
        lg, d = self._distill(student, teacher_values, teacher_indices, teacher_log_sum, labels, temperature,
                              distill_weight, label_weight, vocab)
        (rows, cols), stat = student.shape, _stat_dtype(student.dtype)
        if row_scale is not None:
            _need("row_scale", row_scale, (rows,), stat)
        loss = self._out("loss", loss, (rows,), stat)
        gradient = self._out("gradient", gradient, student.shape, student.dtype)
        self._call(self._lib.pcu_native_distill_step, ctypes.byref(lg), ctypes.byref(d),
                   row_scale.ptr if row_scale is not None else None, loss.ptr, gradient.ptr, cols, cols)
        return loss, gradient

    def native_sample(self, logits: DeviceArray, uniform: DeviceArray, temperature=1.0, top_k=0, top_p=1.0,
                      min_p=0.0, vocab: Optional[int] = None, tokens: Optional[DeviceArray] = None,
                      log_prob: Optional[DeviceArray] = None):
        """One token a row from the row's uniform random number in [0, 1): ``(tokens int32,
        log_prob float32)``. A setting is a number for all rows or an array [rows] (float32,
        ``top_k`` int32); ``temperature`` 0 takes the largest logit, ``top_k`` <= 0 sets no
        limit. The token depends on nothing but the row, its settings and its random number
        (see pcu_native_sample)."""
        lg = self._logits("sample", logits, vocab)
        rows = logits.shape[0]
        _need("uniform", uniform, (rows,), _FLOAT32)
        p = _abi.Sampling(uniform=uniform.ptr)
        for name, x in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
            if isinstance(x, DeviceArray):
                _need(name, x, (rows,), _INT32 if name == "top_k" else _FLOAT32)
                setattr(p, name, x.ptr)
            elif name == "top_k":  # past 31 bits every number sets no limit, as 0 does
                x = operator.index(x)
                p.top_k_value = x if 0 < x < 1 << 31 else 0
            else:
                setattr(p, name + "_value", x)
        tokens = self._out("tokens", tokens, (rows,), _INT32)
        log_prob = self._out("log_prob", log_prob, (rows,), _FLOAT32)
        self._call(self._lib.pcu_native_sample, ctypes.byref(lg), ctypes.byref(p), tokens.ptr, log_prob.ptr)
        return tokens, log_prob

    # ----------------------------------- operators around a model's products
    # Rows are [rows, columns] arrays of float32, float64, float16 or ``bfloat16``, tokens and labels
    # int32 arrays. Results that are not passed in are allocated.
    def _rows(self, what: str, x: DeviceArray) -> _abi.Rows:
        code = _logit_code(what, x.dtype)
        if len(x.shape) != 2:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"{what}: {x.shape} is no array of rows")
        return _abi.Rows(x.ptr, code, 0, x.shape[0], x.shape[1], x.shape[1])

    def native_embedding(self, table: DeviceArray, tokens: DeviceArray, scale: float = 1.0,
                         out: Optional[DeviceArray] = None) -> DeviceArray:
        """``scale`` times the table's row of each token, [tokens, width]; a negative token's row is
        zeros (pcu_native_embedding)."""
        rows = self._rows("embedding", table)
        if len(tokens.shape) != 1:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"embedding: tokens are {tokens.shape}")
        _need("tokens", tokens, tokens.shape, _INT32)
        count, width = tokens.shape[0], table.shape[1]
        out = self._out("out", out, (count, width), table.dtype)
        self._call(self._lib.pcu_native_embedding, ctypes.byref(rows), tokens.ptr, count, scale, out.ptr, width)
        return out

    def native_embedding_backward(self, gradient: DeviceArray, tokens: DeviceArray, table_rows: int,
                                  scale: float = 1.0, base: Optional[DeviceArray] = None,
                                  out: Optional[DeviceArray] = None) -> DeviceArray:
        """The gradient by a table of ``table_rows`` rows: ``base`` (default: zeros; it may be ``out``)
        plus ``scale`` times the sum of each token's rows of ``gradient``, in their order
        (pcu_native_embedding_backward)."""
        rows = self._rows("embedding gradient", gradient)
        count, width = gradient.shape
        table_rows = operator.index(table_rows)
        if not 0 <= table_rows <= _abi.TABLE_MAX_ROWS:
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"embedding gradient: a table of {table_rows} rows")
        _need("tokens", tokens, (count,), _INT32)
        if base is not None:
            _need("base", base, (table_rows, width), gradient.dtype)
        out = self._out("out", out, (table_rows, width), gradient.dtype)
        self._call(self._lib.pcu_native_embedding_backward, ctypes.byref(rows), tokens.ptr, table_rows, scale,
                   base.ptr if base is not None else None, width, out.ptr, width)
        return out

    def _norm_weights(self, x: DeviceArray, weights) -> int:
        """The type's code of the weights among `weights` that there are."""
        dtype = next((w.dtype for w in weights if w is not None), x.dtype)
        if dtype != x.dtype and not (dtype == _FLOAT32 and x.dtype.itemsize == 2):
            raise PcuExecutionError(_abi.PCU_ERR_SHAPE, f"layer_norm: weights of {dtype} for rows of {x.dtype}")
        for w in weights:
            if w is not None:
                _need("weight", w, (x.shape[1],), dtype)
        return _logit_code("layer_norm", dtype)

    def native_layer_norm(self, x: DeviceArray, weight: Optional[DeviceArray] = None,
                          bias: Optional[DeviceArray] = None, eps: float = 1e-5,
                          out: Optional[DeviceArray] = None, stats: Optional[DeviceArray] = None):
        """Layer norm of each row: ``(out, stats)``, ``stats`` [rows, 2] the mean and the reciprocal
        of the standard deviation, as the backward pass takes them. ``weight`` and ``bias`` are of
        the rows' type, or float32 for 16-bit rows; ``out`` may be ``x`` (pcu_native_layer_norm)."""
        rows = self._rows("layer_norm", x)
        code = self._norm_weights(x, (weight, bias))
        out = self._out("out", out, x.shape, x.dtype)
        stats = self._out("stats", stats, (x.shape[0], 2), _stat_dtype(x.dtype))
        self.check(self._lib.pcu_native_layer_norm(
            self.handle, ctypes.byref(rows), weight.ptr if weight is not None else None,
            bias.ptr if bias is not None else None, code, eps, out.ptr, x.shape[1], stats.ptr))
        return out, stats

    def native_layer_norm_backward(self, x: DeviceArray, stats: DeviceArray, gradient: DeviceArray,
                                   weight: Optional[DeviceArray] = None, x_gradient: Optional[DeviceArray] = None,
                                   weight_gradient: Optional[DeviceArray] = None,
                                   bias_gradient: Optional[DeviceArray] = None):
        """The gradients of native_layer_norm from its ``x`` and ``stats``: ``(x_gradient,
        weight_gradient, bias_gradient)``. With a ``weight``, or an array for one of them, the weight's
        and the bias's are computed, else None. ``x_gradient`` may be ``gradient`` or ``x``
        (pcu_native_layer_norm_backward)."""
        rows = self._rows("layer_norm", x)
        width = x.shape[1]
        _need("stats", stats, (x.shape[0], 2), _stat_dtype(x.dtype))
        _need("gradient", gradient, x.shape, x.dtype)
        code = self._norm_weights(x, (weight, weight_gradient, bias_gradient))
        x_gradient = self._out("x_gradient", x_gradient, x.shape, x.dtype)
        if weight is not None:
            weight_gradient = weight_gradient if weight_gradient is not None else self.empty((width,), weight.dtype)
            bias_gradient = bias_gradient if bias_gradient is not None else self.empty((width,), weight.dtype)
        self.check(self._lib.pcu_native_layer_norm_backward(
            self.handle, ctypes.byref(rows), stats.ptr, gradient.ptr, width,
            weight.ptr if weight is not None else None, code, x_gradient.ptr, width,
            weight_gradient.ptr if weight_gradient is not None else None,
            bias_gradient.ptr if bias_gradient is not None else None))
        return x_gradient, weight_gradient, bias_gradient

    def _entropy(self, features: DeviceArray, weights: DeviceArray, labels: DeviceArray, vocab: Optional[int]):
        x, w = self._rows("cross_entropy", features), self._rows("cross_entropy", weights)
        if features.dtype != weights.dtype or features.shape[1] != weights.shape[1] or \
                (vocab is not None and not 0 <= vocab <= weights.shape[0]):
            raise PcuExecutionError(
                _abi.PCU_ERR_SHAPE, f"cross_entropy: features {features.shape} {features.dtype}, weights "
                f"{weights.shape} {weights.dtype}, vocab {vocab}")
        if vocab is not None:
            w.rows = vocab
        _need("labels", labels, (features.shape[0],), _INT32)
        return x, w

    def native_cross_entropy_loss(self, features: DeviceArray, weights: DeviceArray, labels: DeviceArray,
                                  vocab: Optional[int] = None, loss: Optional[DeviceArray] = None,
                                  log_sum: Optional[DeviceArray] = None):
        """Each row's cross entropy of softmax(features * weights^T) against its label (negative:
        none, loss 0), without the logits in memory: ``(loss [rows], log_sum [rows])``, float32.
        ``weights`` holds one row a token; ``vocab`` (default: all) names how many leading rows are
        real. float32, float16 and ``bfloat16`` (pcu_native_cross_entropy_loss)."""
        x, w = self._entropy(features, weights, labels, vocab)
        rows = features.shape[0]
        loss = self._out("loss", loss, (rows,), _FLOAT32)
        log_sum = self._out("log_sum", log_sum, (rows,), _FLOAT32)
        self._call(self._lib.pcu_native_cross_entropy_loss, ctypes.byref(x), ctypes.byref(w), labels.ptr, loss.ptr, log_sum.ptr)
        return loss, log_sum

    def native_cross_entropy_backward(self, features: DeviceArray, weights: DeviceArray, labels: DeviceArray,
                                      log_sum: DeviceArray, row_scale: Optional[DeviceArray] = None,
                                      vocab: Optional[int] = None, feature_gradient: Optional[DeviceArray] = None,
                                      weight_gradient: Optional[DeviceArray] = None):
        """The gradients of the loss, each row times its ``row_scale``, from
        native_cross_entropy_loss's ``log_sum``: ``(feature_gradient, weight_gradient)``, like
        ``features`` and ``weights`` (rows past the vocabulary are 0)."""
        x, w = self._entropy(features, weights, labels, vocab)
        rows, width = features.shape
        _need("log_sum", log_sum, (rows,), _FLOAT32)
        if row_scale is not None:
            _need("row_scale", row_scale, (rows,), _FLOAT32)
        feature_gradient = self._out("feature_gradient", feature_gradient, features.shape, features.dtype)
        weight_gradient = self._out("weight_gradient", weight_gradient, weights.shape, weights.dtype)
        self._call(self._lib.pcu_native_cross_entropy_backward, ctypes.byref(x), ctypes.byref(w), labels.ptr, log_sum.ptr,
                   row_scale.ptr if row_scale is not None else None, feature_gradient.ptr, width, weight_gradient.ptr,
                   weights.shape[0], width)
        return feature_gradient, weight_gradient

    def native_cross_entropy_step(self, features: DeviceArray, weights: DeviceArray, labels: DeviceArray,
                                  row_scale: Optional[DeviceArray] = None, vocab: Optional[int] = None,
                                  loss: Optional[DeviceArray] = None, feature_gradient: Optional[DeviceArray] = None,
                                  weight_gradient: Optional[DeviceArray] = None):
        """native_cross_entropy_loss and native_cross_entropy_backward in one call:
        ``(loss [rows], feature_gradient, weight_gradient)``."""
        x, w = self._entropy(features, weights, labels, vocab)
        rows, width = features.shape
        if row_scale is not None:
            _need("row_scale", row_scale, (rows,), _FLOAT32)
        loss = self._out("loss", loss, (rows,), _FLOAT32)
        feature_gradient = self._out("feature_gradient", feature_gradient, features.shape, features.dtype)
        weight_gradient = self._out("weight_gradient", weight_gradient, weights.shape, weights.dtype)
        self._call(self._lib.pcu_native_cross_entropy_step, ctypes.byref(x), ctypes.byref(w), labels.ptr,
                   row_scale.ptr if row_scale is not None else None, loss.ptr, feature_gradient.ptr, width,
                   weight_gradient.ptr, weights.shape[0], width)
        return loss, feature_gradient, weight_gradient
