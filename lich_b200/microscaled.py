"""Microscaled layers: 8-bit checkpoints of states with the backward products that read them, and 4-bit operands
with their product.

Blocks of 32 numbers share one power of two (formats and layouts: ``include/ipc_b200.h``).  Like the builders of
``lich_b200.tilelang_kernels`` each ``build_*`` returns a cached callable specialised for its shape, activation and
dtype that writes its output tensors in place on the current CUDA stream, raises ``ValueError`` for tensors of another
shape, dtype, device or layout before anything is launched, and holds (per device and stream) whatever workspace it
needs.  Large products with a checkpoint need one of the size of the states in 16 bits; a program that runs many of them in
order passes one buffer of its own instead: ``kernel(..., workspace=buffer)``, ``kernel.workspace_bytes()`` long.  Of a
``KernelConfig`` these products follow ``backend`` (auto, simt, tcgen05) and refuse the rest.

    codes, scales = empty_checkpoint(D, B, device=dev)                       # states x [D, B] kept in 8 bits
    build_checkpoint(D, B, "bfloat16")(x, codes, scales)
    build_checkpoint_restore(D, B, "tanh", "bfloat16")(codes, scales, out)   # out = f(x^)
    build_weight_update_checkpoint(M, K, B, "tanh", "bfloat16", alpha)(w, e, codes, scales)       # W += alpha E f(x^)^T
    build_weight_delta_checkpoint(M, K, B, "tanh", "bfloat16", alpha)(dw, e, codes, scales)       # dW, W untouched
    build_error_backward_checkpoint(M, K, B, "tanh", "bfloat16")(w, e, codes, scales, e_up)       # f'(x^) * (W^T E)

    wq, ws = empty_mxfp4(M, K, device=dev)                                   # weights [M, K] in 4 bits
    build_mxfp4_quantize(M, K, "identity", "bfloat16")(w, wq, ws)
    aq, as_ = empty_mxfp4(B, K, device=dev)                                  # f(x) of states [K, B], turned to [B, K]
    build_mxfp4_quantize(B, K, "tanh", "bfloat16", True)(x, aq, as_)
    build_mxfp4_forward(M, K, B, "bfloat16")(wq, ws, aq, as_, out)           # out [M, B] = W4 @ A4^T

The reference has no counterpart: it keeps and multiplies fp16 only (``tilelang_kernels.py:8-17``).
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import threading
import weakref
from ctypes import byref, c_size_t, c_void_p, cast
from functools import lru_cache, wraps

import torch

from . import _native as N
from .tilelang_kernels import KernelConfig, _algo

N.load()


def _load_call():
    """``csrc/mx_call.cpp``: the checked call in C++ (built beside the library)."""
    path = N.LIB_PATH.parent / "_mx_call.so"
    if not path.exists():
        raise RuntimeError(f"native module {path} is missing: build it with `python -m lich_b200.build`")
    loader = importlib.machinery.ExtensionFileLoader("_mx_call", str(path))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_mx_call", loader))
    loader.exec_module(module)
    return module


_Call = _load_call().Call


class _Scratch:
    """Device memory that operators share, freed when the last one that holds it goes."""

    def __init__(self, n: int, device):
        self.bytes = n
        self._buf = torch.empty(n, device=device, dtype=torch.uint8) if n else None
        self.address = None if self._buf is None else self._buf.data_ptr()


_scratch: weakref.WeakValueDictionary = weakref.WeakValueDictionary()
_ws_lock = threading.Lock()

BLOCK = 32
MAX_SIZE = 2 ** 31 - 512  # of a row or a column: the C entries' sizes, padded to whole tiles, are 32-bit integers
# what torch.cuda.current_device() and current_stream().cuda_stream come down to, at a tenth of their cost
_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def checkpoint_shapes(D: int, B: int) -> tuple[tuple[int, int], tuple[int, int]]:
    """Shapes of a checkpoint's codes (int8) and scale bytes (uint8) for states ``[D, B]``."""
    nb = -(-int(B) // BLOCK)
    return (int(D), nb * BLOCK), (nb, int(D))


def mxfp4_shapes(R: int, K: int) -> tuple[tuple[int, int], tuple[int, ...]]:
    """Shapes of a 4-bit operand's codes and scale bytes (both uint8) for ``R`` rows and ``K`` columns."""
    ka = -(-int(K) // 128)
    return (int(R), ka * 64), (-(-int(R) // 128), ka, 32, 4, 4)


def empty_checkpoint(D: int, B: int, *, device) -> tuple[torch.Tensor, torch.Tensor]:
    c, s = checkpoint_shapes(D, B)
    return torch.empty(c, device=device, dtype=torch.int8), torch.empty(s, device=device, dtype=torch.uint8)


def empty_mxfp4(R: int, K: int, *, device) -> tuple[torch.Tensor, torch.Tensor]:
    c, s = mxfp4_shapes(R, K)
    return torch.empty(c, device=device, dtype=torch.uint8), torch.empty(s, device=device, dtype=torch.uint8)


class _MxOp:
    """Shape-specialised callable over the C ABI: ``spec`` names each tensor argument's shape and dtype."""

    kind = "op"
    call_kind = -1  # the kind and ...
    call_ints: tuple = ()  # ... the attributes that the C++ call passes on as integers
    alpha = 0.0

    def __init__(self, entry: str, spec):
        self.spec = tuple((torch.Size(s), d) for s, d in spec)
        self._fn = getattr(N.load(), entry)
        self._ws: dict = {}
        self._need: int | None = None

    def fast(self):
        """This operator as a C++ callable, which comes back here for everything but a plain call."""
        return _Call(self, self.call_kind, cast(self._fn, c_void_p).value, list(self.spec),
                     tuple(int(getattr(self, n)) for n in self.call_ints), float(self.alpha))

    def _failed(self, rc: int) -> None:
        N.check(rc)

    def _stream(self, tensors):
        """The current stream of the tensors' device, after checking the tensors against ``spec``; None when that device is
        not the current one (``_elsewhere``)."""
        try:
            dev = tensors[0].get_device()
            for t, (shape, dtype) in zip(tensors, self.spec):
                if t.shape != shape or t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
                    break
            else:
                if dev >= 0:
                    return _current_stream(dev) if dev == _current_device() else None
        except (AttributeError, RuntimeError):  # not a tensor; one that cannot be asked for its device or strides
            pass
        raise ValueError(self._refusal(tensors))

    def _elsewhere(self, *tensors, **kw) -> None:
        with torch.cuda.device(tensors[0].device):
            self(*tensors, **kw)

    def _refusal(self, tensors) -> str:
        for i, (t, (shape, dtype)) in enumerate(zip(tensors, self.spec)):
            if not isinstance(t, torch.Tensor):
                return f"{self.kind}: argument {i} is not a tensor"
            if t.shape != shape:
                return f"{self.kind}: argument {i} has shape {tuple(t.shape)}, kernel was built for {tuple(shape)}"
            if t.dtype != dtype:
                return f"{self.kind}: argument {i} is {t.dtype}, kernel was built for {dtype}"
            if not t.is_cuda:
                return f"{self.kind}: argument {i} is not a CUDA tensor"
            if t.layout is not torch.strided:
                return f"{self.kind}: argument {i} is {t.layout}, not a dense tensor"
            if not t.is_contiguous():
                return f"{self.kind}: argument {i} is not contiguous"
        return f"{self.kind}: tensors on different devices"

    def _ws_key(self) -> tuple:
        """What the size of the workspace depends on."""
        raise NotImplementedError

    def _workspace(self, dev: int, stream: int):
        """(address, bytes, owner) of the workspace for one stream of a device: calls on two streams may overlap.
        Operators that differ in what the workspace does not depend on (the factor alpha) share it.  One per stream
        whichever threads ask first; the memory lives as long as an ``owner`` is held, which each operator does."""
        ws = self._ws.get((dev, stream))
        if ws is None:
            with _ws_lock:
                key = self._ws_key() + (dev, stream)
                ws = _scratch.get(key)
                if ws is None:
                    with torch.cuda.device(dev):
                        ws = _Scratch(self.workspace_bytes(), f"cuda:{dev}")
                    _scratch[key] = ws
                self._ws[dev, stream] = ws
        return ws.address, ws.bytes, ws

    def workspace_bytes(self) -> int:
        """Bytes of workspace a call needs (0 for most small shapes)."""
        if self._need is None:
            n = c_size_t(0)
            N.check(self._ws_bytes(byref(n)))
            self._need = int(n.value)
        return self._need

    def _given(self, workspace, dev: int):
        """(address, bytes) of a caller's workspace, after checking it."""
        if not isinstance(workspace, torch.Tensor) or not workspace.is_cuda or workspace.get_device() != dev:
            raise ValueError(f"{self.kind}: the workspace is no tensor on the operands' device")
        if not workspace.is_contiguous():
            raise ValueError(f"{self.kind}: the workspace is not contiguous")
        n, need = workspace.numel() * workspace.element_size(), self.workspace_bytes()
        if n < need or workspace.data_ptr() % 16:
            raise ValueError(f"{self.kind}: a workspace of {n} bytes at {workspace.data_ptr():#x}, {need} bytes needed on a "
                             "16-byte boundary")
        return workspace.data_ptr(), n

    def get_kernel_source(self) -> str:
        return f"lich_b200 {self.kind} {self.spec} (prebuilt sm_100a kernel, include/ipc_b200.h)"


class CheckpointKernel(_MxOp):
    kind = "checkpoint"
    call_kind, call_ints = 0, ("D", "B", "dt")

    def __init__(self, D, B, dtype):
        c, s = checkpoint_shapes(D, B)
        super().__init__("ipc_mx8_store", [((D, B), N.torch_dtype(dtype)), (c, torch.int8), (s, torch.uint8)])
        self.D, self.B, self.dt = int(D), int(B), N.dtype_code(dtype)

    def __call__(self, x, codes, scales):
        s = self._stream((x, codes, scales))
        if s is None:
            return self._elsewhere(x, codes, scales)
        rc = self._fn(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), self.D, self.B, self.dt, s)
        if rc:
            N.check(rc)


class CheckpointRestoreKernel(_MxOp):
    kind = "checkpoint_restore"
    call_kind, call_ints = 1, ("D", "B", "act", "dt")

    def __init__(self, D, B, activation, dtype):
        c, s = checkpoint_shapes(D, B)
        super().__init__("ipc_mx8_restore", [(c, torch.int8), (s, torch.uint8), ((D, B), N.torch_dtype(dtype))])
        self.D, self.B, self.act, self.dt = int(D), int(B), N.act_code(activation), N.dtype_code(dtype)

    def __call__(self, codes, scales, out):
        s = self._stream((codes, scales, out))
        if s is None:
            return self._elsewhere(codes, scales, out)
        rc = self._fn(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), self.D, self.B, self.act, self.dt, s)
        if rc:
            N.check(rc)


class CheckpointWeightKernel(_MxOp):
    kind = "weight_checkpoint"
    call_kind, call_ints = 2, ("mode", "M", "K", "B", "act", "dt", "algo")

    def __init__(self, mode, M, K, B, activation, dtype, alpha, out_dtype, cfg):
        c, s = checkpoint_shapes(K, B)
        dt = N.torch_dtype(dtype)
        super().__init__("ipc_mx8_weight", [((M, K), out_dtype), ((M, B), dt), (c, torch.int8), (s, torch.uint8)])
        self.mode, self.M, self.K, self.B = mode, int(M), int(K), int(B)
        self.act, self.dt, self.alpha, self.algo = N.act_code(activation), N.dtype_code(dtype), float(alpha), _algo(cfg)

    def _ws_key(self) -> tuple:
        return "weight", self.mode, self.M, self.K, self.B, self.dt, self.algo

    def _ws_bytes(self, n) -> int:
        return N.load().ipc_mx8_weight_ws_bytes(self.mode, self.M, self.K, self.B, self.dt, self.algo, n)

    def __call__(self, out, e, codes, scales, *, accumulate: bool = False, workspace=None):
        s = self._stream((out, e, codes, scales))
        if accumulate and self.mode != N.MODE_WDELTA:
            raise ValueError(f"{self.kind}: only a weight delta in float32 accumulates")
        if s is None:
            return self._elsewhere(out, e, codes, scales, accumulate=accumulate, workspace=workspace)
        dev = out.get_device()
        ws, n = self._workspace(dev, s)[:2] if workspace is None else self._given(workspace, dev)
        rc = self._fn(self.mode, out.data_ptr(), e.data_ptr(), codes.data_ptr(), scales.data_ptr(), self.M, self.K, self.B,
                      self.alpha, N.FLAG_ACCUMULATE if accumulate else 0, self.act, self.dt, self.algo, ws, n, s)
        if rc:
            N.check(rc)


class CheckpointBackwardKernel(_MxOp):
    kind = "error_backward_checkpoint"
    call_kind, call_ints = 3, ("M", "K", "B", "act", "dt", "algo")

    def __init__(self, M, K, B, activation, dtype, cfg):
        c, s = checkpoint_shapes(K, B)
        dt = N.torch_dtype(dtype)
        super().__init__("ipc_mx8_backward",
                         [((M, K), dt), ((M, B), dt), (c, torch.int8), (s, torch.uint8), ((K, B), dt)])
        self.M, self.K, self.B = int(M), int(K), int(B)
        self.act, self.dt, self.algo = N.act_code(activation), N.dtype_code(dtype), _algo(cfg)

    def _ws_key(self) -> tuple:
        return "backward", self.M, self.K, self.B, self.dt, self.algo

    def _ws_bytes(self, n) -> int:
        return N.load().ipc_mx8_backward_ws_bytes(self.M, self.K, self.B, self.dt, self.algo, n)

    def __call__(self, w, e, codes, scales, e_up, *, workspace=None):
        s = self._stream((w, e, codes, scales, e_up))
        if s is None:
            return self._elsewhere(w, e, codes, scales, e_up, workspace=workspace)
        dev = w.get_device()
        ws, n = self._workspace(dev, s)[:2] if workspace is None else self._given(workspace, dev)
        rc = self._fn(e_up.data_ptr(), w.data_ptr(), e.data_ptr(), codes.data_ptr(), scales.data_ptr(), self.M, self.K,
                      self.B, self.act, self.dt, self.algo, ws, n, s)
        if rc:
            N.check(rc)


class Mxfp4QuantizeKernel(_MxOp):
    kind = "mxfp4_quantize"
    call_kind, call_ints = 4, ("R", "K", "turned", "act", "dt")

    def __init__(self, R, K, activation, dtype, turned):
        c, s = mxfp4_shapes(R, K)
        super().__init__("ipc_mxfp4_quantize", [((K, R) if turned else (R, K), N.torch_dtype(dtype)),
                                                (c, torch.uint8), (s, torch.uint8)])
        self.R, self.K, self.turned = int(R), int(K), int(bool(turned))
        self.act, self.dt = N.act_code(activation), N.dtype_code(dtype)

    def __call__(self, x, codes, scales):
        s = self._stream((x, codes, scales))
        if s is None:
            return self._elsewhere(x, codes, scales)
        rc = self._fn(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), self.R, self.K, self.turned, self.act, self.dt, s)
        if rc:
            N.check(rc)


class Mxfp4RestoreKernel(_MxOp):
    kind = "mxfp4_restore"
    call_kind, call_ints = 5, ("R", "K", "dt")

    def __init__(self, R, K, dtype):
        c, s = mxfp4_shapes(R, K)
        super().__init__("ipc_mxfp4_restore", [(c, torch.uint8), (s, torch.uint8), ((R, K), N.torch_dtype(dtype))])
        self.R, self.K, self.dt = int(R), int(K), N.dtype_code(dtype)

    def __call__(self, codes, scales, out):
        s = self._stream((codes, scales, out))
        if s is None:
            return self._elsewhere(codes, scales, out)
        rc = self._fn(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), self.R, self.K, self.dt, s)
        if rc:
            N.check(rc)


class Mxfp4ForwardKernel(_MxOp):
    kind = "mxfp4_forward"
    call_kind, call_ints = 6, ("M", "K", "B", "dt")

    def __init__(self, M, K, B, dtype):
        wc, ws = mxfp4_shapes(M, K)
        ac, as_ = mxfp4_shapes(B, K)
        super().__init__("ipc_mxfp4_forward", [(wc, torch.uint8), (ws, torch.uint8), (ac, torch.uint8),
                                               (as_, torch.uint8), ((M, B), N.torch_dtype(dtype))])
        self.M, self.K, self.B, self.dt = int(M), int(K), int(B), N.dtype_code(dtype)

    def __call__(self, w, w_scales, a, a_scales, out):
        s = self._stream((w, w_scales, a, a_scales, out))
        if s is None:
            return self._elsewhere(w, w_scales, a, a_scales, out)
        rc = self._fn(w.data_ptr(), w_scales.data_ptr(), a.data_ptr(), a_scales.data_ptr(), out.data_ptr(), self.M, self.K,
                      self.B, self.dt, s)
        if rc:
            N.check(rc)


def _builder(build):
    """A cached builder of C++ callables."""
    @lru_cache(maxsize=256)
    @wraps(build)
    def cached(*args, **kw):
        return build(*args, **kw).fast()
    return cached


def _validate(*sizes, activation="identity", dtype):
    if min(int(n) for n in sizes) < 0:
        raise ValueError(f"negative size in {sizes}")
    if max(int(n) for n in sizes) > MAX_SIZE:
        raise ValueError(f"a size in {sizes} is above {MAX_SIZE}")
    N.act_code(activation)
    N.dtype_code(N.torch_dtype(dtype))


def _backend(cfg: KernelConfig, dtype) -> None:
    """Refuse what a checkpoint product could only ignore."""
    algo = _algo(cfg)
    if algo == N.ALGO_CODES["outer"]:
        raise ValueError("no outer-product kernel reads checkpoints: backend must be auto, simt or tcgen05")
    if algo == N.ALGO_CODES["tcgen05"] and N.torch_dtype(dtype) is torch.float32:
        raise ValueError("the tensor cores take 16-bit storage: backend tcgen05 is not for float32")
    if cfg.tune() is not None:
        raise ValueError("checkpoint products choose their own tiles, splits and CTAs: of cfg only backend applies (tc_* = 0)")


@_builder
def build_checkpoint(D: int, B: int, dtype: str):
    """``kernel(x [D, B], codes, scales)``: the states in 8 bits."""
    _validate(D, B, dtype=dtype)
    return CheckpointKernel(D, B, dtype)


@_builder
def build_checkpoint_restore(D: int, B: int, activation: str, dtype: str):
    """``kernel(codes, scales, out [D, B])``: ``out = f(x^)``."""
    _validate(D, B, activation=activation, dtype=dtype)
    return CheckpointRestoreKernel(D, B, activation, dtype)


@_builder
def build_weight_update_checkpoint(M: int, K: int, B: int, activation: str, dtype: str, alpha: float,
                                   cfg: KernelConfig = KernelConfig()):
    """``kernel(w [M, K], e [M, B], codes, scales)``: ``W += alpha * E @ f(x^)^T`` in place."""
    _validate(M, K, B, activation=activation, dtype=dtype)
    _backend(cfg, dtype)
    return CheckpointWeightKernel(N.MODE_WEIGHT, M, K, B, activation, dtype, alpha, N.torch_dtype(dtype), cfg)


@_builder
def build_weight_delta_checkpoint(M: int, K: int, B: int, activation: str, dtype: str, alpha: float,
                                  delta_dtype: str = "float32", cfg: KernelConfig = KernelConfig()):
    """``kernel(dw [M, K], e [M, B], codes, scales, accumulate=False)``: ``dw = alpha * E @ f(x^)^T``, in float32 (which
    alone can accumulate) or in ``dtype``."""
    _validate(M, K, B, activation=activation, dtype=dtype)
    _backend(cfg, dtype)
    out = N.torch_dtype(delta_dtype)
    if out is not torch.float32 and out is not N.torch_dtype(dtype):
        raise ValueError(f"a weight delta is kept in float32 or in {dtype}, not in {delta_dtype}")
    mode = N.MODE_WDELTA if out is torch.float32 else N.MODE_WGRAD
    return CheckpointWeightKernel(mode, M, K, B, activation, dtype, alpha, out, cfg)


@_builder
def build_error_backward_checkpoint(M: int, K: int, B: int, activation: str, dtype: str,
                                    cfg: KernelConfig = KernelConfig()):
    """``kernel(w [M, K], e [M, B], codes, scales, e_up [K, B])``: ``e_up = f'(x^) * (W^T @ E)``."""
    _validate(M, K, B, activation=activation, dtype=dtype)
    _backend(cfg, dtype)
    return CheckpointBackwardKernel(M, K, B, activation, dtype, cfg)


@_builder
def build_mxfp4_quantize(R: int, K: int, activation: str, dtype: str, turned: bool = False):
    """``kernel(x, codes, scales)``: ``f(x)`` as a 4-bit operand of ``R`` rows; ``x`` is ``[R, K]``, or with ``turned``
    the feature-major ``[K, R]``."""
    _validate(R, K, activation=activation, dtype=dtype)
    return Mxfp4QuantizeKernel(R, K, activation, dtype, turned)


@_builder
def build_mxfp4_restore(R: int, K: int, dtype: str):
    """``kernel(codes, scales, out [R, K])``: the values a 4-bit operand stands for."""
    _validate(R, K, dtype=dtype)
    return Mxfp4RestoreKernel(R, K, dtype)


@_builder
def build_mxfp4_forward(M: int, K: int, B: int, dtype: str):
    """``kernel(w, w_scales, a, a_scales, out [M, B])``: ``out = W4 @ A4^T``, sums in float32, stored in ``dtype``."""
    _validate(M, K, B, dtype=dtype)
    return Mxfp4ForwardKernel(M, K, B, dtype)
