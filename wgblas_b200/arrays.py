"""Resident typed arrays: ``GpuArray``, and the conversions of its 16-bit types.

``GpuVector`` and ``GpuMatrix`` hold the reference's float32 and float64 data.
The products of language-model layers (``gemmGrouped``, ``mxGemm``, ...) also
take 16-bit floats, index arrays and packed bytes, as flat arrays whose
dimensions and strides are arguments of the call, the way the BLAS routines
take typed arrays. Where they take a ``GpuArray`` they also take a CUDA tensor
of another library that has torch's ``data_ptr`` / ``dtype`` / ``get_device``
interface; it stands for the memory from its first element on.

numpy has no bfloat16: such data is passed and read as uint16 bit patterns
(``toBfloat16`` / ``fromBfloat16`` convert).
"""
from __future__ import annotations

import ctypes as ct

import numpy as np

from . import _native as nat
from ._runtime import Device, Error

_NUMPY = {"float32": np.float32, "bfloat16": np.uint16, "float16": np.float16, "int32": np.int32, "uint8": np.uint8}
_ITEM = {"float32": 4, "bfloat16": 2, "float16": 2, "int32": 4, "uint8": 1}
# WG_TYPE_* codes of the types that products compute with.
TYPE_CODES = {"float32": nat.WG_TYPE_F32, "bfloat16": nat.WG_TYPE_BF16, "float16": nat.WG_TYPE_F16}


def toBfloat16(x) -> np.ndarray:
    """The bfloat16 bit patterns (uint16) of float32 values, rounded to nearest even; NaN stays NaN."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    u = x.view(np.uint32)
    r = ((u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def fromBfloat16(u) -> np.ndarray:
    """The float32 values of bfloat16 bit patterns (uint16)."""
    return (np.ascontiguousarray(u, dtype=np.uint16).astype(np.uint32) << np.uint32(16)).view(np.float32)


class GpuArray:
    """A flat typed array resident in device memory.

    ``dtype`` is "float32", "bfloat16", "float16", "int32" or "uint8".
    """

    __slots__ = ("_buf", "length", "dtype", "device", "ptr", "__weakref__")

    def __init__(self, buffer, length, dtype, device):
        self._buf = buffer
        self.length = length
        self.dtype = dtype
        self.device = device
        p = ct.c_void_p()
        nat.check(nat.lib.wg_buffer_device_ptr(buffer, ct.byref(p)))
        self.ptr = p.value or 0

    @staticmethod
    def empty(device: Device, length: int, dtype: str) -> "GpuArray":
        """An uninitialised array of ``length`` elements."""
        if not isinstance(device, Device) or device.destroyed:
            raise Error("device must be a GPUDevice.")
        if dtype not in _ITEM:
            raise Error("dtype must be one of " + ", ".join(f"'{t}'" for t in _ITEM) + ".")
        if not isinstance(length, (int, np.integer)) or isinstance(length, bool) or length < 0:
            raise Error("length must be a non-negative integer.")
        h = nat.c_buf_p()
        nat.check(nat.lib.wg_buffer_alloc(device.handle, int(length) * _ITEM[dtype], ct.byref(h)))
        return GpuArray(h, int(length), dtype, device)

    @staticmethod
    def from_(device: Device, data: np.ndarray, dtype: str | None = None) -> "GpuArray":
        """Uploads an array (flattened). ``dtype`` defaults to the data's own type; float32
        data is converted when "bfloat16" or "float16" is asked for, uint16 data given
        with "bfloat16" is taken as bit patterns."""
        data = np.asarray(data)
        if dtype is None:
            dtype = next((t for t, n in _NUMPY.items() if data.dtype == n and t != "bfloat16"), None)
        if dtype not in _ITEM:
            raise Error("GpuArray.from expects float32, float16, int32 or uint8 data, or a dtype to hold it in.")
        if dtype == "bfloat16" and data.dtype == np.float32:
            data = toBfloat16(data)
        elif dtype == "float16" and data.dtype == np.float32:
            data = data.astype(np.float16)
        if data.dtype != _NUMPY[dtype]:
            raise Error(f"GpuArray.from cannot hold {data.dtype} data as {dtype}.")
        out = GpuArray.empty(device, data.size, dtype)
        try:
            out.write(data)
        except Exception:
            out.destroy()
            raise
        return out

    def write(self, data: np.ndarray) -> None:
        """Copies ``data`` (the array's type, at most its length) over the array's beginning."""
        self._require_live()
        data = np.ascontiguousarray(data).reshape(-1)
        if data.dtype != _NUMPY[self.dtype] or data.size > self.length:
            raise Error("data must have the array's type and at most its length.")
        nat.check(nat.lib.wg_buffer_upload(self._buf, 0, data.ctypes.data_as(ct.c_void_p), data.nbytes))

    def read(self) -> np.ndarray:
        """The array's elements (bfloat16 as uint16 bit patterns), once the device's queued work is done."""
        self._require_live()
        out = np.empty(self.length, _NUMPY[self.dtype])
        nat.check(nat.lib.wg_buffer_download(self._buf, 0, out.ctypes.data_as(ct.c_void_p), out.nbytes))
        return out

    def destroy(self) -> None:
        if self._buf is not None:
            nat.lib.wg_buffer_free(self._buf)
            self._buf = None
            self.ptr = 0
            self.length = 0

    def _require_live(self):
        if self._buf is None:
            raise Error("GpuArray has been destroyed.")

    def __repr__(self):
        return f"<GpuArray {self.length} {self.dtype} on {self.device!r}>"


setattr(GpuArray, "from", GpuArray.from_)

# dtype objects of other libraries' tensors, by the object: filled as they are met.
_foreign_types: dict = {}


def _foreign_type(dtype):
    name = str(dtype).rsplit(".", 1)[-1]
    _foreign_types[dtype] = name if name in _ITEM else None
    return _foreign_types[dtype]


def resident(device: Device, routine: str, name: str, x):
    """(address, elements from there on, type name) of a GpuArray or CUDA tensor operand on ``device``."""
    if type(x) is GpuArray:
        if x.device is not device:
            raise Error(
                f"{routine}: {name} belongs to a different GPUDevice than the one passed in. "
                "GPU buffers cannot be shared across devices — recreate the operand on this "
                "device, or call the routine with the device that owns it.")
        x._require_live()
        return x.ptr, x.length, x.dtype
    try:
        if not x.is_cuda:
            raise Error(f"{name} must be a GpuArray or a CUDA tensor.")
        ptr, dtype = x.data_ptr(), x.dtype
        if x.get_device() != device.ordinal:
            raise Error(f"{routine}: {name} is on cuda:{x.get_device()}, the device passed in is "
                        f"cuda:{device.ordinal}.")
    except AttributeError:
        raise Error(f"{name} must be a GpuArray or a CUDA tensor.") from None
    kind = _foreign_types[dtype] if dtype in _foreign_types else _foreign_type(dtype)
    if kind is None:
        raise Error(f"{name} has the unsupported type {dtype}.")
    if x.is_contiguous():
        n = x.numel()
    else:  # a strided view: its storage from the first element on
        item = x.element_size()
        n = x.untyped_storage().nbytes() // item - x.storage_offset()
    return ptr, n, kind


def disjoint(name: str, out, out_type: str, others) -> None:
    """Refuses an output whose used elements overlap an operand's: ``out`` and each of
    ``others`` (name, address, elements, type) give the used ranges."""
    p, n = out
    end = p + n * _ITEM[out_type]
    for other, q, m, t in others:
        if n and m and p < q + m * _ITEM[t] and q < end:
            raise Error(f"{name} must not overlap {other}.")
