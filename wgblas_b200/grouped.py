"""``gemmGrouped`` / ``gemmGroupedInner``: matrix products grouped by expert.

Layers that route each row to one of several weight matrices need two products
that a plain gemm does not give. With rows sorted by group and ``offsets`` (groups
+ 1 int32 on the device) naming their ranges:

* ``gemmGrouped``:       C[r] := alpha * A[r] op(B_g) + beta * C[r], r in group g's rows
* ``gemmGroupedInner``:  C_g  := alpha * A[rows of g]^T B[rows of g] + beta * C_g

With weights W_g stored n x k, the layer's forward product is
``gemmGrouped(..., "transpose", ...)``, the gradient of its input
``gemmGrouped(..., "no-transpose", ...)`` on the output's gradient with n and k
exchanged, and the gradient of the weights ``gemmGroupedInner`` of the output's
gradient and the input.

Operands are flat resident arrays (``GpuArray``, or CUDA tensors of another
library) read as row-major matrices; A and B are both bfloat16 or both float16,
C has their type or float32; sums are held in 32 bits. The arguments follow
``sgemm``'s; the reference has no counterpart. Two things differ from ``sgemm``
on resident operands: a call returns when its work is queued on the device's
stream (``GpuArray.read`` or ``device.synchronize()`` waits for it), except on
a benchmark device, which waits and returns ``gpuTimeMs``; and errors that only
the device can see (offsets that decrease or leave the rows: they are clamped) are
raised by ``device.check()``.

CUDA tensors must be ordered on the device's stream: call
``device.set_stream(torch.cuda.current_stream().cuda_stream)`` first. A device's own stream
waits for no work of another library, nor that work for it.
"""
from __future__ import annotations

import ctypes as ct
import math

from . import _native as nat
from ._runtime import Error, require_gpu_device
from .arrays import TYPE_CODES, disjoint, resident
from .classes import _is_int
from .gemm import _TRANS, _is_number


def check_scalars(alpha, beta) -> None:
    for name, v in (("alpha", alpha), ("beta", beta)):
        if type(v) is not float and not _is_number(v):
            raise Error(f"{name} must be a number.")
        if math.isnan(v):
            raise Error(f"{name} must not be NaN.")
        if not math.isfinite(v):
            raise Error(f"{name} must be finite.")


def check_ints(names: str, *values):
    for v in values:
        if type(v) is not int and not _is_int(v):
            raise Error(f"{names} must be integers.")
    return values if all(type(v) is int for v in values) else tuple(int(v) for v in values)


def span(rows: int, cols: int, ld: int) -> int:
    """Elements from a matrix's first to its last, 0 when it has none."""
    return (rows - 1) * ld + cols if rows > 0 and cols > 0 else 0


def need(name: str, have: int, want: int, what: str) -> None:
    if have < want:
        raise Error(f"{name} does not have enough elements for the given {what}.")


def check_offsets(device, routine, offsets, groups: int) -> int:
    ptr, n, kind = resident(device, routine, "offsets", offsets)
    if kind != "int32":
        raise Error("offsets must be int32.")
    need("offsets", n, groups + 1, "groups")
    return ptr


def check_groups(groups: int) -> None:
    if groups > nat.WG_MAX_GROUPS:
        raise Error(f"groups must be at most {nat.WG_MAX_GROUPS}.")


def timed(device, call, *args):
    """Queues a C-ABI call; on a benchmark device waits and returns its gpuTimeMs."""
    if not device.benchmark:
        nat.check(call(*args, None))
        return {}
    ms = ct.c_float(0.0)
    nat.check(call(*args, ct.byref(ms)))
    device.check()
    return {"gpuTimeMs": float(ms.value)}


def gemmGrouped(device, transB, groups, m, n, k, alpha, A, lda, B, ldb, strideB, offsets, beta, C, ldc):
    """C[r] := alpha * A[r] op(B_g) + beta * C[r] for the rows r of each group g.

    A is m x k, C m x n, B_g (``strideB`` elements apart; 0 shares one matrix) k x n for
    "no-transpose" or n x k for "transpose". Rows that no group holds keep their C.
    Queued on the device's stream, on which CUDA tensors must be ordered (``set_stream``).
    """
    st = nat._fast.gemm_grouped(device, transB, groups, m, n, k, alpha, A, lda, B, ldb, strideB, offsets, beta, C, ldc)
    if st is not None:  # the ordinary call, checked and made
        return nat.check(st) or {}
    require_gpu_device(device)
    if transB not in _TRANS:
        raise Error("transB must be 'no-transpose' or 'transpose'.")
    check_scalars(alpha, beta)
    groups, m, n, k, lda, ldb, strideB, ldc = check_ints("groups, m, n, k, lda, ldb, strideB, and ldc", groups, m, n, k,
                                                         lda, ldb, strideB, ldc)
    pa, na, ta = resident(device, "gemmGrouped", "A", A)
    pb, nb, tb = resident(device, "gemmGrouped", "B", B)
    pc, nc, tc = resident(device, "gemmGrouped", "C", C)
    _check_types(ta, tb, tc)
    if groups < 0 or m < 0 or n < 0 or k < 0:
        raise Error("groups, m, n, and k must be non-negative.")
    check_groups(groups)
    if lda <= 0 or ldb <= 0 or ldc <= 0:
        raise Error("lda, ldb, and ldc must be positive.")
    if strideB < 0:
        raise Error("strideB must be non-negative.")
    trans = transB == "transpose"
    rows_b, cols_b = (n, k) if trans else (k, n)
    if lda < k:
        raise Error("lda must be >= cols of A as stored.")
    if ldb < cols_b:
        raise Error("ldb must be >= cols of B as stored.")
    if ldc < n:
        raise Error("ldc must be >= cols of C as stored.")
    po = check_offsets(device, "gemmGrouped", offsets, groups)
    if groups == 0 or m == 0 or n == 0:
        return {}
    use_a, use_b, use_c = span(m, k, lda), span(rows_b, cols_b, ldb), span(m, n, ldc)
    if use_b:
        use_b += (groups - 1) * strideB
    if alpha != 0:
        need("A", na, use_a, "m, k, and lda")
        need("B", nb, use_b, "groups, n, k, ldb, and strideB")
    need("C", nc, use_c, "m, n, and ldc")
    disjoint("C", (pc, use_c), tc, (("A", pa, use_a, ta), ("B", pb, use_b, tb), ("offsets", po, groups + 1, "int32")))
    return timed(device, nat.lib.wg_gemm_grouped_dev, device.handle, TYPE_CODES[ta], TYPE_CODES[tc], int(trans), groups,
                 m, n, k, alpha, pa, lda, pb, ldb, strideB, po, beta, pc, ldc)


def gemmGroupedInner(device, groups, m, n, k, alpha, A, lda, B, ldb, offsets, beta, C, ldc, strideC):
    """C_g := alpha * A[rows of g]^T B[rows of g] + beta * C_g for each group g.

    A is k x m, B k x n, C_g (``strideC`` elements apart) m x n; ``offsets`` groups the k rows.
    A group without rows gives beta * C_g.
    Queued on the device's stream, on which CUDA tensors must be ordered (``set_stream``).
    """
    st = nat._fast.gemm_grouped_inner(device, groups, m, n, k, alpha, A, lda, B, ldb, offsets, beta, C, ldc, strideC)
    if st is not None:
        return nat.check(st) or {}
    require_gpu_device(device)
    check_scalars(alpha, beta)
    groups, m, n, k, lda, ldb, ldc, strideC = check_ints("groups, m, n, k, lda, ldb, ldc, and strideC", groups, m, n, k,
                                                         lda, ldb, ldc, strideC)
    pa, na, ta = resident(device, "gemmGroupedInner", "A", A)
    pb, nb, tb = resident(device, "gemmGroupedInner", "B", B)
    pc, nc, tc = resident(device, "gemmGroupedInner", "C", C)
    _check_types(ta, tb, tc)
    if groups < 0 or m < 0 or n < 0 or k < 0:
        raise Error("groups, m, n, and k must be non-negative.")
    check_groups(groups)
    if lda <= 0 or ldb <= 0 or ldc <= 0:
        raise Error("lda, ldb, and ldc must be positive.")
    if lda < m:
        raise Error("lda must be >= cols of A as stored.")
    if ldb < n:
        raise Error("ldb must be >= cols of B as stored.")
    if ldc < n:
        raise Error("ldc must be >= cols of C as stored.")
    if groups > 1 and strideC < span(m, n, ldc):
        raise Error("strideC must be at least one matrix of C.")
    po = check_offsets(device, "gemmGroupedInner", offsets, groups)
    if groups == 0 or m == 0 or n == 0:
        return {}
    use_a, use_b = span(k, m, lda), span(k, n, ldb)
    use_c = (groups - 1) * strideC + span(m, n, ldc)
    if alpha != 0:
        need("A", na, use_a, "k, m, and lda")
        need("B", nb, use_b, "k, n, and ldb")
    need("C", nc, use_c, "groups, m, n, ldc, and strideC")
    disjoint("C", (pc, use_c), tc, (("A", pa, use_a, ta), ("B", pb, use_b, tb), ("offsets", po, groups + 1, "int32")))
    return timed(device, nat.lib.wg_gemm_grouped_inner_dev, device.handle, TYPE_CODES[ta], TYPE_CODES[tc], groups, m, n,
                 k, alpha, pa, lda, pb, ldb, po, beta, pc, ldc, strideC)


def _check_types(ta, tb, tc) -> None:
    if ta not in ("bfloat16", "float16") or tb != ta:
        raise Error("A and B must both be bfloat16 or both float16.")
    if tc not in (ta, "float32"):
        raise Error("C must have the type of A and B, or float32.")
