"""Device buffers for callers that hand the decoder HBM-resident inputs.

Binds hipMalloc / hipMemcpy / hipFree / hipDeviceSynchronize from the same
libamdhip64 that libparakeet_hip.so links, so pointers stay within one HIP
runtime instance.
"""
from __future__ import annotations

import ctypes as C
import sys

import numpy as np

_hip = None
H2D, D2H, D2D = 1, 2, 3


def hip():
    global _hip
    if _hip is None:
        L = C.CDLL("libamdhip64.so.7")
        L.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
        L.hipFree.argtypes = [C.c_void_p]
        L.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
        L.hipMemset.argtypes = [C.c_void_p, C.c_int, C.c_size_t]
        L.hipGetDevice.argtypes = [C.POINTER(C.c_int)]
        L.hipStreamIsCapturing.argtypes = [C.c_void_p, C.POINTER(C.c_int)]
        L.hipGetErrorString.restype = C.c_char_p
        _hip = L
    return _hip


def _check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what}: {hip().hipGetErrorString(rc).decode()}")


class DeviceArray:
    def __init__(self, nbytes: int):
        self.nbytes = max(int(nbytes), 1)
        p = C.c_void_p()
        _check(hip().hipMalloc(C.byref(p), self.nbytes), "hipMalloc")
        self.ptr = p.value

    @classmethod
    def from_numpy(cls, a: np.ndarray):
        a = np.ascontiguousarray(a)
        d = cls(a.nbytes)
        _check(hip().hipMemcpy(d.ptr, a.ctypes.data, a.nbytes, H2D), "hipMemcpy H2D")
        return d

    def to_numpy(self, dtype, count: int) -> np.ndarray:
        out = np.empty(count, dtype)
        _check(hip().hipMemcpy(out.ctypes.data, self.ptr, out.nbytes, D2H), "hipMemcpy D2H")
        return out

    def zero(self):
        _check(hip().hipMemset(self.ptr, 0, self.nbytes), "hipMemset")

    def free(self):
        if self.ptr:
            hip().hipFree(self.ptr)
            self.ptr = None

    def __del__(self):
        # No HIP call while the interpreter shuts down: the runtime (and a
        # profiler's preloaded library) may already be torn down by then.
        # Callers free their buffers explicitly; a buffer left to the garbage
        # collector at exit is reclaimed with the process.
        if sys.is_finalizing():
            return
        try:
            self.free()
        except Exception:
            pass


NUMPY_TYPES = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "i32": np.int32, "u8": np.uint8}


class Tensor:
    """A device array with a shape, element type ("f32", "f16", "bf16", "i32", "u8") and strides, as
    much of a tensor as the operators of ``lm`` ask for.  bf16 comes and goes as its 16-bit patterns."""

    def __init__(self, shape, dtype: str, buffer: DeviceArray | None = None, offset: int = 0, strides=None):
        self.shape, self.dtype = tuple(int(n) for n in shape), dtype
        self.itemsize = np.dtype(NUMPY_TYPES[dtype]).itemsize
        self.buffer = DeviceArray(self.numel() * self.itemsize) if buffer is None else buffer
        self.offset = offset                      # elements
        if strides is None:
            strides, n = [], 1
            for k in reversed(self.shape):
                strides.insert(0, n)
                n *= k
        self._strides = tuple(strides)

    @classmethod
    def from_numpy(cls, a: np.ndarray, dtype: str | None = None):
        """dtype: only to say that uint16 patterns are bf16 ones."""
        kinds = {np.dtype(v): k for k, v in NUMPY_TYPES.items()}
        a = np.ascontiguousarray(a)
        return cls(a.shape, dtype or kinds[a.dtype], DeviceArray.from_numpy(a))

    def numel(self):
        return int(np.prod(self.shape, dtype=np.int64))

    def data_ptr(self):
        return self.buffer.ptr + self.offset * self.itemsize

    def stride(self):
        return self._strides

    def is_contiguous(self):
        n = 1
        for k, s in zip(reversed(self.shape), reversed(self._strides)):
            if k > 1 and s != n:
                return False
            n *= k
        return True

    def view(self, shape, strides=None, offset: int = 0):
        """The same memory under another shape: strides and offset in elements."""
        return Tensor(shape, self.dtype, self.buffer, self.offset + offset, strides)

    def numpy(self) -> np.ndarray:
        """A host copy, strides followed."""
        kind = NUMPY_TYPES[self.dtype]
        flat = self.buffer.to_numpy(kind, self.buffer.nbytes // self.itemsize)
        return np.lib.stride_tricks.as_strided(flat[self.offset:], self.shape, [s * self.itemsize for s in self._strides]).copy()

    def zero(self):
        self.buffer.zero()


def device() -> int:
    """The current device."""
    d = C.c_int()
    _check(hip().hipGetDevice(C.byref(d)), "hipGetDevice")
    return d.value


def capturing(stream) -> bool:
    """Whether a graph is being captured on the stream."""
    status = C.c_int()
    _check(hip().hipStreamIsCapturing(stream, C.byref(status)), "hipStreamIsCapturing")
    return status.value != 0


def synchronize():
    _check(hip().hipDeviceSynchronize(), "hipDeviceSynchronize")
