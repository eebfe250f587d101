"""Array plumbing between the caller's arrays and the device.

Callers hand the API numpy arrays (as with the reference) or torch tensors.
Kernels only ever see device memory: numpy inputs are copied to the current
CUDA device, torch CUDA tensors are used in place.  Results come back in the
caller's kind: numpy for numpy inputs, a CUDA tensor if any input was on the
device, a (pinned) CPU tensor for CPU tensors.

Element types: the kernels compute in float32 or float64.  float32 features
stay float32 (the B200 path); float64 stays float64 (the reference's own
precision, ``python/mojodgl/_lib.py:127-163``); every other input goes through
the reference's ``f64()`` rules -- complex is rejected, integers that float64
cannot hold exactly are rejected, the rest widen to float64.  Half and bf16
tensors compute in float32, except where an operator takes bf16 as it is
(segment_mm, gather_mm and the operators of a mixture-of-experts layer).
"""

from __future__ import annotations

import numpy as np
import torch

from ._lib import BGL_BF16, BGL_F32, BGL_F64
from .base import DGLError

NUMPY, TORCH_CPU, TORCH_CUDA = 0, 1, 2


_DEVICES = {}  # current device index -> torch.device, filled once a CUDA device has been seen
# the current stream's handle without a Stream object (0.1 us against 3 us)
_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def device() -> torch.device:
    if _DEVICES:
        index = torch.cuda.current_device()
        dev = _DEVICES.get(index)
        if dev is not None:
            return dev
    if not torch.cuda.is_available():
        raise DGLError("mojodgl (B200 build) needs a CUDA device; it has no CPU fallback")
    index = torch.cuda.current_device()
    return _DEVICES.setdefault(index, torch.device("cuda", index))


def stream() -> int:
    if _RAW_STREAM is not None:
        return _RAW_STREAM(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


def kind_of(*xs) -> int:
    k = NUMPY
    for x in xs:
        if isinstance(x, torch.Tensor):
            k = max(k, TORCH_CUDA if x.is_cuda else TORCH_CPU)
    return k


def is_torch(x) -> bool:
    return isinstance(x, torch.Tensor)


# ----------------------------------------------------------------- id arrays
def ids(a):
    """Node ids / segment lengths as int64 (numpy, or torch if given torch).

    Non-integral floats are rejected rather than truncated
    (python/mojodgl/_lib.py:166-180)."""
    if is_torch(a):
        if a.is_floating_point() and a.numel() and not bool((a == a.floor()).all()):
            raise DGLError("node ids and segment lengths must be whole numbers, got {}".format(a.dtype))
        return a.to(torch.int64).contiguous()
    a = np.asanyarray(a)
    if np.issubdtype(a.dtype, np.floating) and a.size:
        if not bool(np.all(a == np.floor(a))):
            raise DGLError("node ids and segment lengths must be whole numbers, got {}".format(a.dtype))
    return np.ascontiguousarray(a, dtype=np.int64)


# ------------------------------------------------------------ feature arrays
def _check_lossless_np(a: np.ndarray) -> None:
    if np.iscomplexobj(a):
        raise DGLError("the kernels are real-valued; complex input is not supported")
    if np.issubdtype(a.dtype, np.integer) and a.dtype != np.int64 and a.size:
        with np.errstate(invalid="ignore"):
            back = a.astype(np.float64).astype(a.dtype)
        if not bool(np.array_equal(back, a)):
            raise DGLError("{} values do not survive the conversion to float64 exactly".format(a.dtype))


def feature(a):
    """A contiguous float32/float64 feature array of the caller's kind."""
    if is_torch(a):
        if a.is_complex():
            raise DGLError("the kernels are real-valued; complex input is not supported")
        if a.dtype in (torch.float32, torch.float64):
            return a.contiguous()
        if a.dtype in (torch.float16, torch.bfloat16):
            return a.to(torch.float32).contiguous()
        if a.dtype != torch.int64 and a.numel() and not a.dtype.is_floating_point:
            back = a.to(torch.float64).to(a.dtype)
            if not bool(torch.equal(back, a)):
                raise DGLError("{} values do not survive the conversion to float64 exactly".format(a.dtype))
        return a.to(torch.float64).contiguous()
    a = np.asanyarray(a)
    if a.dtype == np.float32 or a.dtype == np.float64:
        return np.ascontiguousarray(a)
    _check_lossless_np(a)
    return np.ascontiguousarray(a, dtype=np.float64)


def common_float(*xs):
    """float32 if every present operand is float32, else float64."""
    present = [x for x in xs if x is not None]
    if present and all(str(x.dtype).endswith("float32") for x in present):
        return torch.float32
    return torch.float64


_CODES = {torch.float32: BGL_F32, torch.float64: BGL_F64, torch.bfloat16: BGL_BF16}


def code_of(dtype: torch.dtype) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise DGLError("unsupported element type {}".format(dtype))
    return code


_NP2T = {np.dtype(np.float32): torch.float32, np.dtype(np.float64): torch.float64,
         np.dtype(np.int64): torch.int64, np.dtype(np.int32): torch.int32,
         np.dtype(np.int8): torch.int8}


def to_dev(a, dtype: torch.dtype = None) -> torch.Tensor:
    """The array as a contiguous tensor on the current CUDA device."""
    dev = device()
    if is_torch(a):
        t = a
        if dtype is not None and t.dtype != dtype:
            t = t.to(dtype)
        if t.device != dev:
            t = t.to(dev, non_blocking=t.is_pinned())
        return t.contiguous()
    arr = np.ascontiguousarray(a)
    t = torch.from_numpy(arr) if arr.dtype in _NP2T else torch.from_numpy(arr.astype(np.float64))
    if dtype is not None and t.dtype != dtype:
        t = t.to(dtype)
    return t.to(dev)


def operands(*xs):
    """``kind_of`` the operands, and the operands with a shape and an element
    type each: lists become numpy arrays, an absent one stays None."""
    kind, plain = NUMPY, False
    for x in xs:
        if isinstance(x, torch.Tensor):
            if x.is_cuda:
                kind = TORCH_CUDA
            elif kind == NUMPY:
                kind = TORCH_CPU
        elif x is not None:
            plain = True
    if plain:
        xs = tuple(x if x is None or isinstance(x, torch.Tensor) else np.asanyarray(x) for x in xs)
    return kind, xs


# what ``feature`` makes of arrays of these types, whatever their values
_FEATURE_TYPES = {torch.float32: torch.float32, torch.float64: torch.float64, torch.float16: torch.float32,
                  torch.bfloat16: torch.float32, np.dtype(np.float32): torch.float32,
                  np.dtype(np.float64): torch.float64}


def is_bf16(a) -> bool:
    return isinstance(a, torch.Tensor) and a.dtype == torch.bfloat16


def is_f32(a) -> bool:
    return a.dtype == (torch.float32 if isinstance(a, torch.Tensor) else np.float32)


def float_type(*xs):
    """bfloat16 if every operand is a bfloat16 tensor, else ``common_float`` of
    the operands under the ``feature`` rules."""
    first = getattr(xs[0], "dtype", None)
    if first is torch.bfloat16 or first is torch.float32:  # torch tensors of one such type
        for x in xs:
            if x.dtype is not first:
                break
        else:
            return first
    types = [_FEATURE_TYPES.get(x.dtype) or feature(x).dtype for x in xs]  # (feature checks the others' values)
    return torch.float32 if all(t in (torch.float32, np.float32) for t in types) else torch.float64


def on(dev: torch.device, a, dtype: torch.dtype):
    """``to_dev`` for an operand that may be absent (None), with what is already
    there as asked returned as it is."""
    if a is None:
        return None
    if isinstance(a, torch.Tensor) and a.dtype is dtype and a.device == dev and a.is_contiguous():
        return a
    return to_dev(a, dtype)


def address(t) -> int:
    """Device address of a tensor, None (NULL) for an absent one."""
    return None if t is None else t.data_ptr()


def result(t: torch.Tensor, kind: int):
    """Hand a device result back in the caller's kind."""
    if kind == TORCH_CUDA:
        return t
    if kind == TORCH_CPU:
        out = torch.empty(t.shape, dtype=t.dtype, pin_memory=True)
        out.copy_(t, non_blocking=True)
        torch.cuda.current_stream().synchronize()
        return out
    return t.cpu().numpy()


def ptr(t) -> int:
    """Device address of a tensor, or None (NULL) for an absent/empty one."""
    if t is None or t.numel() == 0:
        return None
    return t.data_ptr()


def workspace(nbytes: int) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device())


def shape_of(a):
    return tuple(a.shape)


def reshape(a, shape):
    return a.reshape(shape)


def zeros_like_kind(shape, dtype, kind):
    if kind == NUMPY:
        return np.zeros(shape, dtype=np.float32 if dtype == torch.float32 else np.float64)
    dev = device() if kind == TORCH_CUDA else "cpu"
    return torch.zeros(shape, dtype=dtype, device=dev)
