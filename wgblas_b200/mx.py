"""Microscaled 4-bit floating point (OCP MXFP4): ``GpuMxMatrix``, ``mxQuantize``,
``mxDequantize``, ``mxGemm`` and ``mxGemmGrouped``.

In MXFP4, 32 neighbouring elements of a row share a power-of-two scale and each
element is one of 0, .5, 1, 1.5, 2, 3, 4, 6 or its negative: 4.25 bits an element. The
tensor cores multiply two matrices quantised along the contraction:

    wq = GpuMxMatrix.empty(device, n, k)                     # weights, once
    mxQuantize(device, "no-transpose", n, k, W, k, wq)
    xq = GpuMxMatrix.empty(device, m, k)                     # activations, each step
    mxQuantize(device, "no-transpose", m, k, X, k, xq)
    mxGemm(device, m, n, k, 1.0, xq, wq, 0.0, Y, n)          # Y = Xq Wq^T

Gradients contract the other dimensions, so they quantise their operands along
those: dX = quantise(dY) quantise(W^T)^T and dW = quantise(dY^T) quantise(X^T)^T, with
"transpose" for the second ones. For rows grouped by expert, ``mxQuantize`` takes
the groups' ``offsets`` and ``mxGemmGrouped`` multiplies by a batch of matrices; the
gradient of grouped weights, whose contraction is ragged, is ``gemmGroupedInner``'s.

Like ``gemmGrouped``, the calls take flat resident arrays read as row-major
matrices, are queued on the device's stream, on which CUDA tensors must be ordered
(``device.set_stream``), and report what only the device can see (bad offsets) at
``device.check()``. The reference has no counterpart.
"""
from __future__ import annotations

import numpy as np

from . import _native as nat
from ._runtime import Device, Error, require_gpu_device
from .arrays import TYPE_CODES, GpuArray, _foreign_types, disjoint, resident
from .gemm import _TRANS
from .grouped import check_groups, check_ints, check_offsets, check_scalars, need, span, timed


def mxCodesSize(rows: int, cols: int, batch: int = 1) -> int:
    """Bytes of the codes of ``batch`` quantised rows x cols matrices."""
    return batch * rows * (-(-cols // 32) * 16)


def mxScalesSize(rows: int, cols: int, batch: int = 1, groups: int = 0) -> int:
    """Bytes of their scales (with ``groups``, of one matrix whose rows are grouped)."""
    return (batch * -(-rows // 128) + groups) * -(-cols // 128) * 512


class GpuMxMatrix:
    """A resident MXFP4 matrix, a batch of them, or one whose rows are grouped.

    ``codes`` and ``scales`` are uint8 ``GpuArray``s or CUDA tensors in the layout of
    include/wgblas.h: rows of two elements a byte, and tiles of 128 rows x 4 scale bytes.
    """

    __slots__ = ("device", "rows", "cols", "batch", "groups", "codes", "scales", "_codes", "_scales", "_owned")

    def __init__(self, device, codes, scales, rows, cols, batch, groups):
        self.device = device
        self.rows, self.cols, self.batch, self.groups = rows, cols, batch, groups
        self.codes, self.scales = codes, scales
        self._codes, nc, tc = resident(device, "GpuMxMatrix", "codes", codes)
        self._scales, ns, ts = resident(device, "GpuMxMatrix", "scales", scales)
        if tc != "uint8" or ts != "uint8":
            raise Error("codes and scales must be uint8.")
        need("codes", nc, mxCodesSize(rows, cols, batch), "rows, cols, and batch")
        need("scales", ns, mxScalesSize(rows, cols, batch, groups), "rows, cols, batch, and groups")
        disjoint("codes", (self._codes, mxCodesSize(rows, cols, batch)), tc,
                 (("scales", self._scales, mxScalesSize(rows, cols, batch, groups), ts),))
        if (self._codes | self._scales) & 15:
            raise Error("codes and scales must be 16-byte aligned.")

    @staticmethod
    def _check(device, rows, cols, batch, groups):
        require_gpu_device(device)
        rows, cols, batch, groups = check_ints("rows, cols, batch, and groups", rows, cols, batch, groups)
        if rows < 0 or cols < 0 or batch < 0 or groups < 0:
            raise Error("rows, cols, batch, and groups must be non-negative.")
        check_groups(groups)
        if groups and batch != 1:
            raise Error("a matrix with grouped rows has batch 1.")
        return rows, cols, batch, groups

    @staticmethod
    def empty(device, rows, cols, batch=1, groups=0) -> "GpuMxMatrix":
        """An uninitialised matrix for ``mxQuantize`` to fill; ``groups`` > 0 for grouped rows."""
        rows, cols, batch, groups = GpuMxMatrix._check(device, rows, cols, batch, groups)
        codes = GpuArray.empty(device, mxCodesSize(rows, cols, batch), "uint8")
        try:
            scales = GpuArray.empty(device, mxScalesSize(rows, cols, batch, groups), "uint8")
        except Exception:
            codes.destroy()
            raise
        x = GpuMxMatrix(device, codes, scales, rows, cols, batch, groups)
        x._owned = True
        return x

    @staticmethod
    def wrap(device, codes, scales, rows, cols, batch=1, groups=0) -> "GpuMxMatrix":
        """A matrix in memory the caller owns."""
        x = nat._fast.mx_wrap(device, codes, scales, rows, cols, batch, groups)
        if x is not None:
            return x
        return GpuMxMatrix(device, codes, scales, *GpuMxMatrix._check(device, rows, cols, batch, groups))

    def destroy(self) -> None:
        """Frees arrays made by ``empty`` (wrapped memory is the caller's)."""
        if getattr(self, "_owned", False):  # (only ``empty`` sets it)
            self.codes.destroy()
            self.scales.destroy()
        self._codes = self._scales = 0
        self.rows = self.cols = 0

    def __repr__(self):
        more = f" batch={self.batch}" if self.batch != 1 else f" groups={self.groups}" if self.groups else ""
        return f"<GpuMxMatrix {self.rows}x{self.cols}{more} on {self.device!r}>"


def _mx(device, routine, name, x, rows, cols):
    if not isinstance(x, GpuMxMatrix):
        raise Error(f"{name} must be a GpuMxMatrix.")
    if x.device is not device:
        raise Error(
            f"{routine}: {name} belongs to a different GPUDevice than the one passed in. "
            "GPU buffers cannot be shared across devices — recreate the operand on this "
            "device, or call the routine with the device that owns it.")
    for part in (x.codes, x.scales):
        if type(part) is GpuArray:
            part._require_live()
    if x.rows != rows or x.cols != cols:
        raise Error(f"{name} is {x.rows} x {x.cols}, the call needs {rows} x {cols}.")


def _grouping(device, routine, x, offsets):
    """The address of ``offsets``, which a matrix with grouped rows needs and no other takes."""
    if x.groups:
        if offsets is None:
            raise Error("a matrix with grouped rows needs offsets.")
        return check_offsets(device, routine, offsets, x.groups)
    if offsets is not None:
        raise Error("offsets need a GpuMxMatrix with groups.")
    return None


def _mx_ranges(x):
    return (("codes", x._codes, mxCodesSize(x.rows, x.cols, x.batch), "uint8"),
            ("scales", x._scales, mxScalesSize(x.rows, x.cols, x.batch, x.groups), "uint8"))


def _offsets_range(x, ptr):
    return (("offsets", ptr, x.groups + 1, "int32"),) if x.groups else ()


def mxQuantize(device, trans, rows, cols, X, ldx, out, offsets=None, strideX=0):
    """out := op(X) in MXFP4; out is rows x cols, its blocks of 32 run along its rows.

    X (float32, bfloat16 or float16) is stored rows x cols for "no-transpose", cols x rows
    for "transpose"; the matrices of a batch are ``strideX`` elements apart (by default one
    after the other). For each block the scale is 2^(floor(log2 max|x|) - 2), at least
    2^-127; elements are rounded to nearest, ties to even, beyond 6 scales to 6. A block
    with a NaN or an infinity becomes NaN.
    Queued on the device's stream, on which CUDA tensors must be ordered (``set_stream``).
    """
    st = nat._fast.mx_quantize(device, trans, rows, cols, X, ldx, out, offsets, strideX)
    if st is not None:  # the ordinary call, checked and made
        return nat.check(st) or {}
    require_gpu_device(device)
    if trans not in _TRANS:
        raise Error("trans must be 'no-transpose' or 'transpose'.")
    rows, cols, ldx, strideX = check_ints("rows, cols, ldx, and strideX", rows, cols, ldx, strideX)
    _mx(device, "mxQuantize", "out", out, rows, cols)
    px, nx, tx = resident(device, "mxQuantize", "X", X)
    if tx not in TYPE_CODES:
        raise Error("X must be float32, bfloat16 or float16.")
    t = trans == "transpose"
    srows, scols = (cols, rows) if t else (rows, cols)
    if ldx <= 0:
        raise Error("ldx must be positive.")
    if ldx < scols:
        raise Error("ldx must be >= cols of X as stored.")
    if strideX < 0:
        raise Error("strideX must be non-negative.")
    if t and out.groups:
        raise Error("grouped rows are quantised without transpose.")
    po = _grouping(device, "mxQuantize", out, offsets)
    if not strideX and out.batch > 1:
        strideX = srows * ldx
    used = span(srows, scols, ldx)
    if not used or not out.batch:
        return {}
    used += (out.batch - 1) * strideX
    need("X", nx, used, "rows, cols, ldx, and strideX")
    for name, p, n, kind in _mx_ranges(out):
        disjoint("out", (p, n), kind, (("X", px, used, tx), *_offsets_range(out, po)))
    return timed(device, nat.lib.wg_mx_quantize_dev, device.handle, TYPE_CODES[tx], int(t), out.batch, rows, cols, px, ldx,
                 strideX, out.groups, po, out._codes, out._scales)


def mxDequantize(device, x, out, ldo, offsets=None, strideO=0):
    """out (rows x cols, ``ldo``; float32, bfloat16 or float16) := the values ``x`` stands for.

    The matrices of a batch go ``strideO`` elements apart (by default one after the
    other). Rows that no group holds are not written.
    Queued on the device's stream, on which CUDA tensors must be ordered (``set_stream``).
    """
    st = nat._fast.mx_dequantize(device, x, out, ldo, offsets, strideO)
    if st is not None:
        return nat.check(st) or {}
    require_gpu_device(device)
    if not isinstance(x, GpuMxMatrix):
        raise Error("x must be a GpuMxMatrix.")
    rows, cols = x.rows, x.cols
    ldo, strideO = check_ints("ldo and strideO", ldo, strideO)
    _mx(device, "mxDequantize", "x", x, rows, cols)
    po, no, to = resident(device, "mxDequantize", "out", out)
    if to not in TYPE_CODES:
        raise Error("out must be float32, bfloat16 or float16.")
    if ldo <= 0:
        raise Error("ldo must be positive.")
    if ldo < cols:
        raise Error("ldo must be >= cols of out as stored.")
    off = _grouping(device, "mxDequantize", x, offsets)
    if not strideO and x.batch > 1:
        strideO = rows * ldo
    used = span(rows, cols, ldo)
    if not used or not x.batch:
        return {}
    if x.batch > 1 and strideO < used:
        raise Error("strideO must be at least one matrix of out.")
    used += (x.batch - 1) * strideO
    need("out", no, used, "rows, cols, ldo, and strideO")
    disjoint("out", (po, used), to, (*_mx_ranges(x), *_offsets_range(x, off)))
    return timed(device, nat.lib.wg_mx_dequantize_dev, device.handle, TYPE_CODES[to], x.batch, rows, cols, x._codes,
                 x._scales, x.groups, off, po, ldo, strideO)


def _product(device, routine, m, n, k, alpha, A, B, beta, C, ldc, groups):
    require_gpu_device(device)
    check_scalars(alpha, beta)
    m, n, k, ldc = check_ints("m, n, k, and ldc", m, n, k, ldc)
    if m < 0 or n < 0 or k < 0:
        raise Error("m, n, and k must be non-negative.")
    _mx(device, routine, "A", A, m, k)
    _mx(device, routine, "B", B, n, k)
    if A.batch != 1 or A.groups != groups or B.groups or B.batch != (groups or 1):
        raise Error("A must have batch 1 and grouped rows, B one matrix for each group." if groups else
                    "A and B must each be one matrix without groups.")
    pc, nc, tc = resident(device, routine, "C", C)
    if tc not in TYPE_CODES:
        raise Error("C must be float32, bfloat16 or float16.")
    if ldc <= 0:
        raise Error("ldc must be positive.")
    if ldc < n:
        raise Error("ldc must be >= cols of C as stored.")
    used = span(m, n, ldc)
    if used:
        need("C", nc, used, "m, n, and ldc")
        disjoint("C", (pc, used), tc, (("A", A._codes, mxCodesSize(m, k), "uint8"),
                                       ("B", B._codes, mxCodesSize(n, k, B.batch), "uint8"),
                                       ("A", A._scales, mxScalesSize(m, k, 1, groups), "uint8"),
                                       ("B", B._scales, mxScalesSize(n, k, B.batch), "uint8")))
    return m, n, k, ldc, pc, tc, used


def mxGemm(device, m, n, k, alpha, A, B, beta, C, ldc):
    """C := alpha * A B^T + beta * C with A (m x k) and B (n x k) in MXFP4.

    C is float32, bfloat16 or float16; sums are held in 32 bits.
    Queued on the device's stream, on which CUDA tensors must be ordered (``set_stream``).
    """
    st = nat._fast.mx_gemm(device, 0, m, n, k, alpha, A, B, None, beta, C, ldc)
    if st is not None:
        return nat.check(st) or {}
    m, n, k, ldc, pc, tc, used = _product(device, "mxGemm", m, n, k, alpha, A, B, beta, C, ldc, 0)
    if not used:
        return {}
    return timed(device, nat.lib.wg_mx_gemm_dev, device.handle, TYPE_CODES[tc], m, n, k, alpha, A._codes, A._scales,
                 B._codes, B._scales, beta, pc, ldc)


def mxGemmGrouped(device, groups, m, n, k, alpha, A, B, offsets, beta, C, ldc):
    """C[r] := alpha * A[r] B_g^T + beta * C[r] for the rows r of each group g.

    A is m x k with rows grouped by ``offsets`` (quantised with the same ones), B a batch
    of ``groups`` n x k matrices. Rows that no group holds keep their C.
    Queued on the device's stream, on which CUDA tensors must be ordered (``set_stream``).
    """
    if groups:
        st = nat._fast.mx_gemm(device, groups, m, n, k, alpha, A, B, offsets, beta, C, ldc)
        if st is not None:
            return nat.check(st) or {}
    (groups,) = check_ints("groups", groups)
    if groups < 0:
        raise Error("groups must be non-negative.")
    check_groups(groups)
    if groups == 0:
        require_gpu_device(device)
        return {}
    m, n, k, ldc, pc, tc, used = _product(device, "mxGemmGrouped", m, n, k, alpha, A, B, beta, C, ldc, groups)
    po = check_offsets(device, "mxGemmGrouped", offsets, groups)
    if not used:
        return {}
    disjoint("C", (pc, used), tc, _offsets_range(A, po))
    return timed(device, nat.lib.wg_mx_gemm_grouped_dev, device.handle, TYPE_CODES[tc], groups, m, n, k, alpha, A._codes,
                 A._scales, B._codes, B._scales, po, beta, pc, ldc)


nat._fast.setup(Device, GpuArray, GpuMxMatrix, _foreign_types)


def mxDecode(codes: np.ndarray, scales: np.ndarray, rows: int, cols: int) -> np.ndarray:
    """The float64 values of one quantised matrix read back to the host (``codes`` and
    ``scales`` as ``GpuArray.read`` gives them)."""
    lut = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
    lut = np.concatenate([lut, -lut])
    c = np.asarray(codes)[: mxCodesSize(rows, cols)].reshape(rows, -1)
    q = lut[np.stack([c & 15, c >> 4], -1)].reshape(rows, -1)[:, :cols]
    tall, wide = -(-rows // 128), -(-cols // 128)
    e = np.asarray(scales)[: mxScalesSize(rows, cols)].reshape(tall, wide, 32, 4, 4).transpose(0, 3, 2, 1, 4)
    e = np.repeat(e.reshape(tall * 128, wide * 4)[:rows], 32, 1)[:, :cols].astype(np.int64)
    return np.where(e == 255, np.nan, np.ldexp(q, e - 127))
