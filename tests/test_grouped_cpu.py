"""Host side of the grouped and MXFP4 products: conversions, storage sizes, the
refusals of every entry point (Python functions, their C fast path, C ABI).
CPU only: a stand-in device whose zero compute capability stops a call that
passes every check with WG_ERR_NOT_SUPPORTED, before any CUDA call."""
from __future__ import annotations

import ctypes as ct

import numpy as np
import pytest

import mx_check as mc

T, N = "transpose", "no-transpose"


class Tensor:
    """A CUDA tensor's interface over an address that is never read."""

    is_cuda = True

    def __init__(self, n, dtype, ptr=1 << 20, device=0, contiguous=True):
        self.n, self.dtype, self.ptr, self.device_index, self.contiguous = n, dtype, ptr, device, contiguous

    def data_ptr(self):
        return self.ptr

    def get_device(self):
        return self.device_index

    def is_contiguous(self):
        return self.contiguous

    def numel(self):
        return self.n

    def element_size(self):
        return {"float32": 4, "int32": 4, "uint8": 1}.get(self.dtype, 2)

    def storage_offset(self):
        return 0

    def untyped_storage(self):
        t = self

        class S:
            def nbytes(self):
                return t.n * t.element_size()

        return S()


def at(i):
    return (i + 1) << 32  # far apart


@pytest.fixture()
def dev(wg):
    block = (ct.c_char * 65536)()
    d = wg.Device(ct.cast(block, ct.c_void_p), 0, False, {}, "stand-in")
    d_keep.append(block)
    return d


d_keep = []


def reached(wg, fn, *args, **kw):
    """The call passes every check (and stops at the device's architecture)."""
    with pytest.raises(wg._native.NativeError) as e:
        fn(*args, **kw)
    assert e.value.status == wg._native.WG_ERR_NOT_SUPPORTED


# ---- gemmGrouped ---------------------------------------------------------------

G, M, NN, K = 3, 10, 6, 8


def grouped_args(wg, dev, **kw):
    a = dict(device=dev, transB=T, groups=G, m=M, n=NN, k=K, alpha=1.0, A=Tensor(M * K, "bfloat16", at(0)), lda=K,
             B=Tensor(G * NN * K, "bfloat16", at(1)), ldb=K, strideB=NN * K, offsets=Tensor(G + 1, "int32", at(2)),
             beta=0.0, C=Tensor(M * NN, "bfloat16", at(3)), ldc=NN)
    a.update(kw)
    return list(a.values())


GROUPED_BAD = [
    (dict(device=None), "device must be a GPUDevice."),
    (dict(transB="yes"), "transB must be"),
    (dict(alpha="1"), "alpha must be a number."),
    (dict(alpha=float("nan")), "alpha must not be NaN."),
    (dict(beta=float("inf")), "beta must be finite."),
    (dict(m=1.5), "must be integers."),
    (dict(ldc=None), "must be integers."),
    (dict(A=np.zeros(80, np.float32)), "A must be a GpuArray or a CUDA tensor."),
    (dict(A=Tensor(80, "float64")), "A has the unsupported type"),
    (dict(A=Tensor(80, "float32")), "A and B must both be bfloat16 or both float16."),
    (dict(B=Tensor(144, "float16", at(1))), "A and B must both be bfloat16 or both float16."),
    (dict(C=Tensor(60, "float16", at(3))), "C must have the type of A and B, or float32."),
    (dict(A=Tensor(80, "bfloat16", at(0), device=1)), "A is on cuda:1"),
    (dict(groups=-1), "must be non-negative."),
    (dict(k=-1), "must be non-negative."),
    (dict(groups=1025, offsets=Tensor(1026, "int32", at(2))), "groups must be at most 1024."),
    (dict(ldb=0), "lda, ldb, and ldc must be positive."),
    (dict(strideB=-1), "strideB must be non-negative."),
    (dict(lda=K - 1), "lda must be >= cols of A as stored."),
    (dict(ldb=K - 1), "ldb must be >= cols of B as stored."),
    (dict(transB=N, ldb=NN - 1), "ldb must be >= cols of B as stored."),
    (dict(ldc=NN - 1), "ldc must be >= cols of C as stored."),
    (dict(offsets=Tensor(G + 1, "uint8", at(2))), "offsets must be int32."),
    (dict(offsets=Tensor(G, "int32", at(2))), "offsets does not have enough elements"),
    (dict(A=Tensor(M * K - 1, "bfloat16", at(0))), "A does not have enough elements"),
    (dict(B=Tensor(G * NN * K - 1, "bfloat16", at(1))), "B does not have enough elements"),
    (dict(strideB=NN * K + 1), "B does not have enough elements"),
    (dict(C=Tensor(M * NN - 1, "bfloat16", at(3))), "C does not have enough elements"),
    (dict(C=Tensor(M * NN, "bfloat16", at(0) + 2 * M * K - 2)), "C must not overlap A."),
    (dict(C=Tensor(M * NN, "bfloat16", at(1) - 2)), "C must not overlap B."),
]


def test_grouped_valid_calls_reach_the_library(wg, dev):
    reached(wg, wg.gemmGrouped, *grouped_args(wg, dev))
    for kw in (dict(transB=N, ldb=NN), dict(strideB=0), dict(C=Tensor(M * NN, "float32", at(3))), dict(beta=2, alpha=3),
               dict(alpha=0.0, beta=0.5, A=Tensor(0, "bfloat16", at(0))), dict(k=0, lda=8, beta=0.5),
               dict(A=Tensor(M * K, "bfloat16", at(0), contiguous=False)), dict(C=Tensor(M * NN, "bfloat16", at(0) + 2 * M * K)),
               dict(m=np.int64(M)), dict(lda=K + 1, A=Tensor((M - 1) * (K + 1) + K, "bfloat16", at(0)))):
        reached(wg, wg.gemmGrouped, *grouped_args(wg, dev, **kw))


@pytest.mark.parametrize("kw,text", GROUPED_BAD, ids=[str(i) for i in range(len(GROUPED_BAD))])
def test_grouped_refusals(wg, dev, kw, text):
    args = grouped_args(wg, dev, **kw)
    assert wg._native._fast.gemm_grouped(*args) is None
    with pytest.raises(wg.Error) as e:
        wg.gemmGrouped(*args)
    assert text in str(e.value)


def test_grouped_nothing_to_do(wg, dev):
    for kw in (dict(m=0), dict(n=0), dict(groups=0)):
        assert wg.gemmGrouped(*grouped_args(wg, dev, **kw)) == {}
    # C stays as it is
    assert wg._native.lib.wg_gemm_grouped_dev(dev.handle, 1, 1, 1, G, 0, NN, K, 1.0, None, K, None, K, 48, None, 0.0, None,
                                              NN, None) == 0


# ---- gemmGroupedInner ------------------------------------------------------------


def inner_args(wg, dev, **kw):
    a = dict(device=dev, groups=G, m=NN, n=K, k=M, alpha=1.0, A=Tensor(M * NN, "float16", at(0)), lda=NN,
             B=Tensor(M * K, "float16", at(1)), ldb=K, offsets=Tensor(G + 1, "int32", at(2)), beta=0.0,
             C=Tensor(G * NN * K, "float32", at(3)), ldc=K, strideC=NN * K)
    a.update(kw)
    return list(a.values())


INNER_BAD = [
    (dict(device=1), "device must be a GPUDevice."),
    (dict(alpha=None), "alpha must be a number."),
    (dict(strideC=0.5), "must be integers."),
    (dict(B=Tensor(80, "bfloat16", at(1))), "A and B must both be"),
    (dict(C=Tensor(144, "bfloat16", at(3))), "C must have the type of A and B, or float32."),
    (dict(n=-2), "must be non-negative."),
    (dict(lda=0), "must be positive."),
    (dict(lda=NN - 1), "lda must be >= cols of A as stored."),
    (dict(ldb=K - 1), "ldb must be >= cols of B as stored."),
    (dict(ldc=K - 1), "ldc must be >= cols of C as stored."),
    (dict(strideC=NN * K - 1), "strideC must be at least one matrix of C."),
    (dict(offsets=Tensor(G, "int32", at(2))), "offsets does not have enough elements"),
    (dict(A=Tensor(M * NN - 1, "float16", at(0))), "A does not have enough elements"),
    (dict(B=Tensor(M * K - 1, "float16", at(1))), "B does not have enough elements"),
    (dict(C=Tensor(G * NN * K - 1, "float32", at(3))), "C does not have enough elements"),
    (dict(C=Tensor(G * NN * K, "float32", at(1) - 4)), "C must not overlap B."),
]


def test_inner_valid_calls_reach_the_library(wg, dev):
    reached(wg, wg.gemmGroupedInner, *inner_args(wg, dev))
    reached(wg, wg.gemmGroupedInner, *inner_args(wg, dev, groups=1, strideC=0))
    reached(wg, wg.gemmGroupedInner, *inner_args(wg, dev, k=0))  # writes zeros


@pytest.mark.parametrize("kw,text", INNER_BAD, ids=[str(i) for i in range(len(INNER_BAD))])
def test_inner_refusals(wg, dev, kw, text):
    args = inner_args(wg, dev, **kw)
    assert wg._native._fast.gemm_grouped_inner(*args) is None
    with pytest.raises(wg.Error) as e:
        wg.gemmGroupedInner(*args)
    assert text in str(e.value)


# ---- MXFP4 ------------------------------------------------------------------------


def mx(wg, dev, rows, cols, batch=1, groups=0, base=10):
    return wg.GpuMxMatrix.wrap(dev, Tensor(wg.mxCodesSize(rows, cols, batch), "uint8", at(base)),
                               Tensor(wg.mxScalesSize(rows, cols, batch, groups), "uint8", at(base + 1)), rows, cols, batch,
                               groups)


def test_mx_sizes(wg):
    assert wg.mxCodesSize(3, 33) == 3 * 32 and wg.mxCodesSize(3, 32, 2) == 2 * 3 * 16
    assert wg.mxScalesSize(129, 129) == 2 * 2 * 512 and wg.mxScalesSize(5, 4, 3) == 3 * 512
    assert wg.mxScalesSize(130, 4, groups=4) == (2 + 4) * 512
    for rows, cols, cuts in ((300, 200, None), (300, 200, [0, 1, 1, 130, 300])):
        code, scale = mc.quantize(np.ones((rows, cols)))
        assert mc.pack_codes(code).size == wg.mxCodesSize(rows, cols)
        have = mc.tile_scales(scale, cuts).size
        if cuts is None:
            assert have == wg.mxScalesSize(rows, cols)
        else:
            assert have <= wg.mxScalesSize(rows, cols, groups=len(cuts) - 1)


@pytest.mark.parametrize("kw,text", [
    (dict(rows=-1), "must be non-negative."), (dict(groups=2, batch=3), "a matrix with grouped rows has batch 1."),
    (dict(rows=2.5), "must be integers."), (dict(groups=2000), "groups must be at most 1024."),
    (dict(rows=101), "codes does not have enough elements"), (dict(groups=1), "scales does not have enough elements"),
    (dict(codes=Tensor(100 * 16, "int32", at(1))), "codes and scales must be uint8."),
    (dict(codes=Tensor(100 * 16, "uint8", at(1) + 8)), "codes and scales must be 16-byte aligned."),
    (dict(device=None), "device must be a GPUDevice."),
])
def test_mx_matrix_refusals(wg, dev, kw, text):
    a = dict(device=dev, codes=Tensor(100 * 16, "uint8", at(1)), scales=Tensor(512, "uint8", at(2)), rows=100, cols=32,
             batch=1, groups=0)
    wg.GpuMxMatrix.wrap(**a)
    a.update(kw)
    with pytest.raises(wg.Error) as e:
        wg.GpuMxMatrix.wrap(**a)
    assert text in str(e.value)


def quant_args(wg, dev, **kw):
    a = dict(device=dev, trans=N, rows=40, cols=50, X=Tensor(2000, "bfloat16", at(0)), ldx=50, out=mx(wg, dev, 40, 50),
             offsets=None, strideX=0)
    a.update(kw)
    return list(a.values())


def test_quantize_checks(wg, dev):
    reached(wg, wg.mxQuantize, *quant_args(wg, dev))
    reached(wg, wg.mxQuantize, *quant_args(wg, dev, trans=T, ldx=40))
    reached(wg, wg.mxQuantize, *quant_args(wg, dev, out=mx(wg, dev, 40, 50, batch=3), X=Tensor(6000, "float32", at(0))))
    reached(wg, wg.mxQuantize, *quant_args(wg, dev, out=mx(wg, dev, 40, 50, groups=2), offsets=Tensor(3, "int32", at(5))))
    for kw, text in (
            (dict(trans=0), "trans must be"), (dict(out=None), "out must be a GpuMxMatrix."),
            (dict(out=mx(wg, dev, 41, 50)), "out is 41 x 50, the call needs 40 x 50."),
            (dict(X=Tensor(2000, "int32", at(0))), "X must be float32, bfloat16 or float16."),
            (dict(ldx=0), "ldx must be positive."), (dict(ldx=49), "ldx must be >= cols of X as stored."),
            (dict(trans=T, ldx=39), "ldx must be >= cols of X as stored."), (dict(strideX=-1), "strideX must be non-negative."),
            (dict(X=Tensor(1999, "bfloat16", at(0))), "X does not have enough elements"),
            (dict(out=mx(wg, dev, 40, 50, batch=2)), "X does not have enough elements"),
            (dict(out=mx(wg, dev, 40, 50, groups=2)), "a matrix with grouped rows needs offsets."),
            (dict(offsets=Tensor(3, "int32", at(5))), "offsets need a GpuMxMatrix with groups."),
            (dict(out=mx(wg, dev, 40, 50, groups=2), offsets=Tensor(2, "int32", at(5))), "offsets does not have enough"),
            (dict(trans=T, ldx=40, out=mx(wg, dev, 40, 50, groups=2), offsets=Tensor(3, "int32", at(5))),
             "grouped rows are quantised without transpose."),
            (dict(X=Tensor(2000, "bfloat16", at(10) + 16)), "out must not overlap X.")):
        args = quant_args(wg, dev, **kw)
        assert wg._native._fast.mx_quantize(*args) is None
        with pytest.raises(wg.Error) as e:
            wg.mxQuantize(*args)
        assert text in str(e.value), (kw, str(e.value))
    assert wg.mxQuantize(*quant_args(wg, dev, rows=0, out=mx(wg, dev, 0, 50))) == {}


def test_dequantize_checks(wg, dev):
    base = dict(device=dev, x=mx(wg, dev, 40, 50), out=Tensor(2000, "float32", at(0)), ldo=50, offsets=None, strideO=0)
    reached(wg, wg.mxDequantize, *base.values())
    for kw, text in ((dict(x=3), "x must be a GpuMxMatrix."), (dict(out=Tensor(2000, "uint8", at(0))), "out must be float32"),
                     (dict(ldo=0), "ldo must be positive."), (dict(ldo=49), "ldo must be >= cols of out as stored."),
                     (dict(out=Tensor(1999, "float32", at(0))), "out does not have enough elements"),
                     (dict(x=mx(wg, dev, 40, 50, batch=2), strideO=1999, out=Tensor(9999, "float32", at(0))),
                      "strideO must be at least one matrix of out."),
                     (dict(x=mx(wg, dev, 40, 50, groups=1)), "a matrix with grouped rows needs offsets."),
                     (dict(out=Tensor(2000, "float32", at(11))), "out must not overlap scales.")):
        args = list({**base, **kw}.values())
        assert wg._native._fast.mx_dequantize(*args) is None
        with pytest.raises(wg.Error) as e:
            wg.mxDequantize(*args)
        assert text in str(e.value), (kw, str(e.value))


def test_mx_gemm_checks(wg, dev):
    base = dict(device=dev, m=40, n=30, k=50, alpha=1.0, A=mx(wg, dev, 40, 50), B=mx(wg, dev, 30, 50, base=12), beta=0.0,
                C=Tensor(1200, "bfloat16", at(0)), ldc=30)
    reached(wg, wg.mxGemm, *base.values())
    reached(wg, wg.mxGemm, *{**base, "alpha": 2, "C": Tensor(1200, "float32", at(0))}.values())
    bad = [(dict(A=None), "A must be a GpuMxMatrix."), (dict(B=mx(wg, dev, 30, 51, base=12)), "B is 30 x 51"),
           (dict(k=-1), "must be non-negative."), (dict(alpha=float("inf")), "alpha must be finite."),
           (dict(A=mx(wg, dev, 40, 50, groups=2)), "A and B must each be one matrix without groups."),
           (dict(B=mx(wg, dev, 30, 50, batch=2, base=12)), "A and B must each be one matrix without groups."),
           (dict(C=Tensor(1200, "int32", at(0))), "C must be float32"), (dict(ldc=0), "ldc must be positive."),
           (dict(ldc=29), "ldc must be >= cols of C as stored."), (dict(C=Tensor(1199, "bfloat16", at(0))), "C does not have"),
           (dict(C=Tensor(1200, "bfloat16", at(13))), "C must not overlap B.")]
    for kw, text in bad:
        a = {**base, **kw}
        assert wg._native._fast.mx_gemm(a["device"], 0, a["m"], a["n"], a["k"], a["alpha"], a["A"], a["B"], None, a["beta"],
                                        a["C"], a["ldc"]) is None
        with pytest.raises(wg.Error) as e:
            wg.mxGemm(*a.values())
        assert text in str(e.value), (kw, str(e.value))
    grouped = dict(device=dev, groups=2, m=40, n=30, k=50, alpha=1.0, A=mx(wg, dev, 40, 50, groups=2),
                   B=mx(wg, dev, 30, 50, batch=2, base=12), offsets=Tensor(3, "int32", at(5)), beta=0.0,
                   C=Tensor(1200, "bfloat16", at(0)), ldc=30)
    reached(wg, wg.mxGemmGrouped, *grouped.values())
    for kw, text in ((dict(A=mx(wg, dev, 40, 50)), "A must have batch 1 and grouped rows"),
                     (dict(B=mx(wg, dev, 30, 50, batch=3, base=12)), "B one matrix for each group"),
                     (dict(offsets=Tensor(2, "int32", at(5))), "offsets does not have enough"), (dict(groups=-1), "non-negative"),
                     (dict(groups=3), "A must have batch 1 and grouped rows")):
        with pytest.raises(wg.Error) as e:
            wg.mxGemmGrouped(*{**grouped, **kw}.values())
        assert text in str(e.value), (kw, str(e.value))
    assert wg.mxGemmGrouped(*{**grouped, "groups": 0}.values()) == {}


def test_codes_and_scales_in_the_same_memory_are_refused(wg, dev):
    codes, scales = wg.mxCodesSize(40, 50), wg.mxScalesSize(40, 50)
    c = Tensor(codes, "uint8", at(0))
    for where in (at(0), at(0) + codes - 16, at(0) - scales + 16):
        with pytest.raises(wg.Error, match="codes must not overlap scales"):
            wg.GpuMxMatrix.wrap(dev, c, Tensor(scales, "uint8", where), 40, 50)
    for where in (at(0) + codes, at(0) - scales):
        wg.GpuMxMatrix.wrap(dev, c, Tensor(scales, "uint8", where), 40, 50)


# ---- C ABI -------------------------------------------------------------------------


def test_abi_refusals(wg, dev):
    L, bad, h = wg._native.lib, wg._native.WG_ERR_INVALID_ARGUMENT, dev.handle
    p = ct.c_void_p(1 << 20)
    odd = ct.c_void_p((1 << 20) + 1)
    ok = [h, 1, 1, 1, 2, 4, 4, 8, 1.0, p, 8, p, 8, 32, p, 0.0, p, 4, None]
    assert L.wg_gemm_grouped_dev(*ok) == wg._native.WG_ERR_NOT_SUPPORTED
    for i, v in ((0, None), (1, 0), (1, 7), (2, 2), (3, 2), (4, -1), (4, 2000), (5, 1 << 31), (6, -1), (9, None), (9, odd),
                 (10, 7), (12, 7), (13, -1), (14, None), (16, None), (16, odd), (17, 3), (17, 1 << 41)):
        a = list(ok)
        a[i] = v
        assert L.wg_gemm_grouped_dev(*a) == bad, (i, v)
    ok = [h, 1, 0, 2, 4, 4, 8, 1.0, p, 8, p, 8, p, 0.0, p, 4, 16, None]
    assert L.wg_gemm_grouped_inner_dev(*ok) == wg._native.WG_ERR_NOT_SUPPORTED
    for i, v in ((0, None), (1, 0), (2, 2), (3, 1025), (8, odd), (9, 3), (11, 3), (12, None), (14, ct.c_void_p((1 << 20) + 2)),
                 (15, 3), (16, 15)):
        a = list(ok)
        a[i] = v
        assert L.wg_gemm_grouped_inner_dev(*a) == bad, (i, v)
    ok = [h, 1, 0, 1, 4, 40, p, 40, 0, 0, None, p, p, None]
    assert L.wg_mx_quantize_dev(*ok) == wg._native.WG_ERR_NOT_SUPPORTED
    for i, v in ((0, None), (1, 5), (2, 2), (3, -1), (5, 1 << 31), (6, None), (7, 39), (8, -1), (9, 2), (11, None),
                 (11, ct.c_void_p((1 << 20) + 8)), (12, None)):
        a = list(ok)
        a[i] = v
        assert L.wg_mx_quantize_dev(*a) == bad, (i, v)
    ok = [h, 1, 1, 4, 40, p, p, 0, None, p, 40, 0, None]
    assert L.wg_mx_dequantize_dev(*ok) == wg._native.WG_ERR_NOT_SUPPORTED
    for i, v in ((0, None), (1, 9), (5, None), (9, None), (10, 39), (2, 2)):
        a = list(ok)
        a[i] = v
        assert L.wg_mx_dequantize_dev(*a) == bad, (i, v)
    ok = [h, 0, 4, 4, 64, 1.0, p, p, p, p, 0.0, p, 4, None]
    assert L.wg_mx_gemm_dev(*ok) == wg._native.WG_ERR_NOT_SUPPORTED
    for i, v in ((0, None), (1, 4), (2, -1), (4, 1 << 31), (6, None), (7, ct.c_void_p((1 << 20) + 4)), (11, None), (12, 3)):
        a = list(ok)
        a[i] = v
        assert L.wg_mx_gemm_dev(*a) == bad, (i, v)
    assert L.wg_mx_gemm_grouped_dev(h, 0, 2, 4, 4, 64, 1.0, p, p, p, p, None, 0.0, p, 4, None) == bad
    assert b"NULL" in L.wg_last_error()


def test_abi_refuses_what_is_not_aligned_to_its_elements(wg, dev):
    """Every pointer of every entry point, one at a time; the kernels read and write whole elements."""
    L, h = wg._native.lib, dev.handle
    p, at1, at2 = (ct.c_void_p((1 << 20) + o) for o in (0, 1, 2))
    f32, bf16 = wg._native.WG_TYPE_F32, wg._native.WG_TYPE_BF16
    calls = [
        (L.wg_gemm_grouped_dev, [h, bf16, bf16, 1, 2, 4, 4, 8, 1.0, p, 8, p, 8, 32, p, 0.0, p, 4, None],
         [(9, at1), (11, at1), (14, at2), (16, at1)]),
        (L.wg_gemm_grouped_inner_dev, [h, bf16, f32, 2, 4, 4, 8, 1.0, p, 8, p, 8, p, 0.0, p, 4, 16, None],
         [(8, at1), (10, at1), (12, at2), (14, at2)]),
        (L.wg_mx_quantize_dev, [h, bf16, 0, 1, 4, 40, p, 40, 0, 2, p, p, p, None], [(6, at1), (10, at2)]),
        (L.wg_mx_quantize_dev, [h, f32, 1, 1, 4, 40, p, 40, 0, 0, None, p, p, None], [(6, at2)]),
        (L.wg_mx_dequantize_dev, [h, f32, 1, 4, 40, p, p, 2, p, p, 40, 0, None], [(8, at1), (9, at2)]),
        (L.wg_mx_gemm_dev, [h, f32, 4, 4, 64, 1.0, p, p, p, p, 0.0, p, 4, None], [(11, at2)]),
        (L.wg_mx_gemm_grouped_dev, [h, bf16, 2, 4, 4, 64, 1.0, p, p, p, p, p, 0.0, p, 4, None], [(11, at2), (13, at1)]),
    ]
    for fn, ok, odd in calls:
        assert fn(*ok) == wg._native.WG_ERR_NOT_SUPPORTED, fn.__name__
        for i, v in odd:
            a = list(ok)
            a[i] = v
            assert fn(*a) == wg._native.WG_ERR_INVALID_ARGUMENT, (fn.__name__, i)
            assert b"aligned to its elements" in L.wg_last_error()


def test_abi_strides_past_64_bits(wg, dev):
    """Matrices that would overlap are refused also where rows * ld leaves 64 bits."""
    L, bad, h = wg._native.lib, wg._native.WG_ERR_INVALID_ARGUMENT, dev.handle
    p, ld = ct.c_void_p(1 << 20), (1 << 40) - 8
    rows = (1 << 24) + 2  # (rows - 1) * ld is 2^64 and a little: 2^40 in 64 bits
    assert L.wg_mx_dequantize_dev(h, 1, 2, rows, 40, p, p, 0, None, p, ld, (1 << 40) - 1, None) == bad
    assert b"at least one matrix" in L.wg_last_error()
    assert L.wg_gemm_grouped_inner_dev(h, 1, 0, 2, rows, 40, 8, 1.0, p, rows, p, 40, p, 0.0, p, ld, (1 << 40) - 1,
                                       None) == bad
    assert b"at least one matrix" in L.wg_last_error()


# ---- conversions -----------------------------------------------------------------------


def test_bfloat16_conversions(wg):
    rng = np.random.default_rng(0)
    x = rng.standard_normal(4096).astype(np.float32) * np.exp2(rng.integers(-130, 120, 4096)).astype(np.float32)
    y = wg.fromBfloat16(wg.toBfloat16(x)).astype(np.float64)
    step = np.exp2(np.maximum(np.floor(np.log2(np.abs(x.astype(np.float64)) + 1e-300)), -126) - 7)
    assert (np.abs(y - x) <= step / 2).all()
    ties = np.array([0x3F808000, 0x3F818000, 0x7F7FFFFF, 0x7F800000, 0xFF800000, 0x7FC00001, 0x7F800001, 0x80000000],
                    np.uint32).view(np.float32)
    assert list(wg.toBfloat16(ties)) == [0x3F80, 0x3F82, 0x7F80, 0x7F80, 0xFF80, 0x7FC0, 0x7FC0, 0x8000]


def test_mx_reference_is_the_definition():
    """tests/mx_check.py against a loop over the definition, at ties and extremes."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 70)) * np.exp2(rng.integers(-6, 6, (6, 70)))
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7]
    x[1, :32] = 0
    x[2, 3] = 1e-45
    x[3, 64] = np.inf
    code, scale = mc.quantize(x)
    for r in range(6):
        for b in range(3):
            blk = x[r, b * 32:(b + 1) * 32]
            if not np.isfinite(blk).all():
                assert scale[r, b] == 255
                continue
            top = np.abs(blk).max()
            e = -127
            while e < 127 and top >= 2.0 ** (e + 1 + 2):
                e += 1
            assert scale[r, b] == e + 127
            for i, v in enumerate(blk):
                a = abs(v) / 2.0 ** e
                d = np.abs(mc.GRID - a)
                near = np.flatnonzero(d == d.min())
                want = near[0] if len(near) == 1 else next(k for k in near if k % 2 == 0)
                assert code[r, b * 32 + i] == want + (8 if np.signbit(v) else 0)


def test_mx_decode_reads_the_storage(wg):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((150, 70))
    code, scale = mc.quantize(x)
    got = wg.mxDecode(mc.pack_codes(code).reshape(-1), mc.tile_scales(scale), 150, 70)
    assert np.array_equal(got, mc.values(code, scale, 70))
