"""gemmGrouped / gemmGroupedInner on the GPU against plain 64-bit products."""
from __future__ import annotations

import numpy as np
import pytest

import grouped_check as gc

pytestmark = pytest.mark.gpu

T, N = "transpose", "no-transpose"


def up(wg, x, dtype):
    """(stored array, the values it holds in float64) of x in a type."""
    x = np.asarray(x, np.float32)
    if dtype == "bfloat16":
        s = wg.toBfloat16(x)
        return s, wg.fromBfloat16(s).astype(np.float64).reshape(x.shape)
    s = x.astype(np.float16 if dtype == "float16" else np.float32)
    return s, s.astype(np.float64)


def values(wg, arr):
    a = arr.read()
    return (wg.fromBfloat16(a) if arr.dtype == "bfloat16" else a).astype(np.float64)


def matrix(rng, outer, rows, cols, ld, extra=0):
    """outer matrices of rows x cols values with leading dimension ld; the padding is NaN."""
    stride = rows * ld + extra
    x = np.full(outer * stride, np.nan, np.float32)
    for g in range(outer):
        for r in range(rows):
            x[g * stride + r * ld:g * stride + r * ld + cols] = rng.standard_normal(cols)
    return x, stride


def view(x, outer, rows, cols, ld, stride):
    return np.lib.stride_tricks.as_strided(x, (outer, rows, cols), (stride * x.itemsize, ld * x.itemsize, x.itemsize))


def run_rows(wg, device, trans, sizes, n, k, dtype="bfloat16", ctype=None, alpha=1.0, beta=0.0, pad=(0, 0, 0, 0),
             first=0, after=0, shift=0, seed=1, share=False):
    """One rows-form call; every element of C's storage is checked. pad: extra lda, ldb, strideB, ldc.
    shift: elements by which every operand is moved off its allocation's start."""
    rng = np.random.default_rng(seed)
    ctype = ctype or dtype
    groups = len(sizes)
    offsets = first + np.concatenate([[0], np.cumsum(sizes)])
    m = int(offsets[-1]) + after
    lda, ldc = k + pad[0], n + pad[3]
    br, bc = (n, k) if trans == T else (k, n)
    ldb = bc + pad[1]
    ax, _ = matrix(rng, 1, m, k, lda)
    bx, strideB = matrix(rng, 1 if share else groups, br, bc, ldb, pad[2])
    if share:
        strideB = 0
    cx, _ = matrix(rng, 1, m, n, ldc)
    put = lambda x: np.concatenate([np.full(shift, np.nan, np.float32), x])  # noqa: E731
    sa, va = up(wg, put(ax), dtype)
    sb, vb = up(wg, put(bx), dtype)
    sc, vc = up(wg, put(cx), ctype)
    va, vb, vc = va[shift:], vb[shift:], vc[shift:]
    A, B, C = (wg.GpuArray.from_(device, s, t) for s, t in ((sa, dtype), (sb, dtype), (sc, ctype)))
    off = wg.GpuArray.from_(device, offsets.astype(np.int32))

    class At:  # a resident operand that begins `shift` elements into an allocation
        is_cuda = True

        def __init__(self, arr):
            self.arr, self.dtype = arr, arr.dtype

        def data_ptr(self):
            return self.arr.ptr + shift * {"float32": 4}.get(self.arr.dtype, 2)

        def get_device(self):
            return device.ordinal

        def is_contiguous(self):
            return True

        def numel(self):
            return self.arr.length - shift

    ops = [At(x) if shift else x for x in (A, B, C)]
    wg.gemmGrouped(device, trans, groups, m, n, k, alpha, ops[0], lda, ops[1], ldb, strideB, off, beta, ops[2], ldc)
    device.check()
    got = values(wg, C)[shift:]
    a = view(va, 1, m, k, lda, 0)[0]
    b = view(vb, groups, br, bc, ldb, strideB)
    c = view(vc, 1, m, n, ldc, 0)[0].copy()
    want, mag = gc.rows_form(a, b, trans == T, offsets, alpha, beta, c)
    gc.assert_close(view(got, 1, m, n, ldc, 0)[0], want, mag, k, beta, c, ctype, "C")
    if ldc > n:  # the padding between rows is never written
        assert np.isnan(view(got, 1, m, ldc, ldc, 0)[0][:, n:]).all()
    for x in (A, B, C, off):
        x.destroy()
    return got


SIZES = [[1], [16], [5, 0, 11], [0, 0, 130, 1, 0], [300, 257], [64] * 9, [1] * 40, [1000, 3]]


@pytest.mark.parametrize("trans", [T, N])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}g{sum(s)}")
@pytest.mark.parametrize("n,k", [(128, 64), (200, 136), (8, 512), (520, 72)])
def test_rows_aligned(wg, device, trans, sizes, n, k):
    run_rows(wg, device, trans, sizes, n, k)


@pytest.mark.parametrize("trans", [T, N])
@pytest.mark.parametrize("sizes", [[3], [7, 0, 150], [1] * 33, [260]], ids=lambda s: f"{len(s)}g{sum(s)}")
@pytest.mark.parametrize("n,k", [(1, 1), (129, 63), (33, 777), (257, 2), (65, 130)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_rows_odd(wg, device, trans, sizes, n, k, dtype):
    run_rows(wg, device, trans, sizes, n, k, dtype)


@pytest.mark.parametrize("dtype,ctype", [("bfloat16", "float32"), ("float16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (0.5, 1.0), (-2.0, 0.25), (0.0, 0.0), (0.0, -1.5), (0.0, 1.0)])
def test_rows_scalars_and_types(wg, device, dtype, ctype, alpha, beta):
    run_rows(wg, device, T, [40, 0, 90], 136, 200, dtype, ctype, alpha, beta)
    run_rows(wg, device, N, [40, 0, 90], 135, 201, dtype, ctype, alpha, beta)


@pytest.mark.parametrize("trans", [T, N])
@pytest.mark.parametrize("pad", [(8, 16, 24, 5), (3, 1, 7, 0), (0, 0, 1, 2), (0, 8, 8, 8)])
def test_rows_strides(wg, device, trans, pad):
    run_rows(wg, device, trans, [33, 70], 136, 200, pad=pad)


@pytest.mark.parametrize("trans", [T, N])
@pytest.mark.parametrize("shift", [1, 2, 4, 8])
def test_rows_alignment_of_the_bases(wg, device, trans, shift):
    run_rows(wg, device, trans, [33, 70], 136, 200, shift=shift)
    run_rows(wg, device, trans, [33, 70], 136, 199, "float16", "float32", beta=1.0, shift=shift)


@pytest.mark.parametrize("trans", [T, N])
def test_rows_of_no_group_stay(wg, device, trans):
    run_rows(wg, device, trans, [20, 0, 15], 136, 72, first=3, after=9)
    run_rows(wg, device, trans, [0, 0], 136, 72, first=3, after=9)


def test_rows_share_one_matrix(wg, device):
    run_rows(wg, device, T, [20, 0, 150], 136, 72, share=True)
    run_rows(wg, device, N, [20, 0, 150], 136, 72, share=True)


def test_rows_most_groups(wg, device):
    run_rows(wg, device, T, [g % 3 for g in range(1024)], 16, 64)


def test_rows_longer_contraction_and_many_tiles(wg, device):
    run_rows(wg, device, T, [700, 1, 900], 1000, 2048)
    run_rows(wg, device, N, [700, 1, 900], 1000, 2048, "float16", "float32")


# Enough tiles, and rows a group, for the CTA-pair form (256 x 256 tiles).
WIDE = [150, 0, 1, 290, 256, 257, 31, 140, 513, 160, 64, 130, 129, 200, 300]


@pytest.mark.parametrize("trans", [T, N])
@pytest.mark.parametrize("n,k", [(2048, 72), (2056, 136), (1800, 200)])
@pytest.mark.parametrize("ctype", ["bfloat16", "float32"])
def test_rows_pairs(wg, device, trans, n, k, ctype):
    run_rows(wg, device, trans, WIDE, n, k, ctype=ctype, first=1, after=5)
    run_rows(wg, device, trans, WIDE, n, k, ctype=ctype, alpha=0.5, beta=-1.0, pad=(8, 16, 24, 3))


def test_rows_pairs_long(wg, device):
    run_rows(wg, device, T, [700, 300], 9600, 2048, ctype="float32")
    run_rows(wg, device, N, [700, 300], 9600, 2056, "float16")


@pytest.mark.parametrize("trans", [T, N])
@pytest.mark.parametrize("sizes,n,k", [([3], 200, 2048), ([1], 128, 8200), ([32, 0, 1, 33, 7], 520, 1030), ([64, 50], 136, 4096),
                                       ([40, 0, 70], 264, 3000), ([17] * 12, 264, 600), ([5], 1024, 65), ([70], 136, 100)])
@pytest.mark.parametrize("ctype", ["bfloat16", "float32"])
def test_rows_split_contraction(wg, device, trans, sizes, n, k, ctype):
    """Few tiles and a long contraction: several CTAs share a tile."""
    run_rows(wg, device, trans, sizes, n, k, ctype=ctype, first=1, after=2)
    run_rows(wg, device, trans, sizes, n, k, ctype=ctype, alpha=0.5, beta=-1.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_odd_many_tiles_and_long(wg, device, dtype):
    run_rows(wg, device, T, [700, 300], 1001, 2049, dtype, "float32")
    run_rows(wg, device, N, [700, 1, 300], 1001, 1999, dtype)


def run_inner(wg, device, sizes, m, n, dtype="bfloat16", ctype="float32", alpha=1.0, beta=0.0, pad=(0, 0, 0, 0), first=0,
              after=0, seed=2, poison=None):
    rng = np.random.default_rng(seed)
    groups = len(sizes)
    offsets = first + np.concatenate([[0], np.cumsum(sizes)])
    k = int(offsets[-1]) + after
    lda, ldb, ldc = m + pad[0], n + pad[1], n + pad[2]
    ax, _ = matrix(rng, 1, k, m, lda)
    bx, _ = matrix(rng, 1, k, n, ldb)
    cx, strideC = matrix(rng, groups, m, n, ldc, pad[3])
    if poison is not None:  # rows of no group hold values that would show in any sum
        for x, ld in ((ax, lda), (bx, ldb)):
            r = x.reshape(k, ld)
            r[:first] = poison
            r[offsets[-1]:] = poison
    sa, va = up(wg, ax, dtype)
    sb, vb = up(wg, bx, dtype)
    sc, vc = up(wg, cx, ctype)
    A, B, C = (wg.GpuArray.from_(device, s, t) for s, t in ((sa, dtype), (sb, dtype), (sc, ctype)))
    off = wg.GpuArray.from_(device, offsets.astype(np.int32))
    wg.gemmGroupedInner(device, groups, m, n, k, alpha, A, lda, B, ldb, off, beta, C, ldc, strideC)
    device.check()
    got = values(wg, C)
    a, b = view(va, 1, k, m, lda, 0)[0], view(vb, 1, k, n, ldb, 0)[0]
    c = view(vc, groups, m, n, ldc, strideC).copy()
    want, mag = gc.inner_form(a, b, offsets, alpha, beta, c)
    gc.assert_close(view(got, groups, m, n, ldc, strideC), want, mag, max(sizes) if sizes else 0, beta, c, ctype, "C")
    if ldc > n:
        assert np.isnan(view(got, groups, m, ldc, ldc, strideC)[..., n:]).all()
    for x in (A, B, C, off):
        x.destroy()


@pytest.mark.parametrize("sizes", SIZES + [[17, 63, 65, 2], [0, 0, 0]], ids=lambda s: f"{len(s)}g{sum(s)}")
@pytest.mark.parametrize("m,n", [(128, 64), (8, 136), (264, 392)])
def test_inner_aligned(wg, device, sizes, m, n):
    run_inner(wg, device, sizes, m, n)


@pytest.mark.parametrize("sizes", [[3], [7, 0, 150], [1] * 33, [260]], ids=lambda s: f"{len(s)}g{sum(s)}")
@pytest.mark.parametrize("m,n", [(1, 1), (129, 63), (33, 301), (257, 2)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_inner_odd(wg, device, sizes, m, n, dtype):
    run_inner(wg, device, sizes, m, n, dtype)


@pytest.mark.parametrize("dtype,ctype", [("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (0.5, 1.0), (-2.0, 0.25), (0.0, 0.0), (0.0, -1.5)])
def test_inner_scalars_and_types(wg, device, dtype, ctype, alpha, beta):
    run_inner(wg, device, [40, 0, 90], 136, 200, dtype, ctype, alpha, beta)


@pytest.mark.parametrize("pad", [(8, 16, 5, 3), (3, 1, 0, 0), (0, 0, 7, 9)])
def test_inner_strides(wg, device, pad):
    run_inner(wg, device, [33, 0, 70], 136, 200, pad=pad)


@pytest.mark.parametrize("m,n", [(520, 776), (264, 1288), (512, 1024)])
@pytest.mark.parametrize("ctype", ["bfloat16", "float32"])
def test_inner_pairs(wg, device, m, n, ctype):
    sizes = [150, 0, 1, 17, 63, 64, 65, 512, 513, 530, 128, 1100, 16, 31, 700, 5]
    run_inner(wg, device, sizes, m, n, ctype=ctype, first=2, after=3, poison=np.nan)
    run_inner(wg, device, sizes, m, n, ctype=ctype, alpha=0.5, beta=1.0, pad=(8, 16, 3, 5))


def test_inner_split_contraction(wg, device):
    run_inner(wg, device, [3000], 136, 264, first=1, after=2, poison=np.nan)
    run_inner(wg, device, [1500, 0, 40, 777], 130, 200, ctype="bfloat16", alpha=0.5, beta=1.0)
    run_inner(wg, device, [129], 64, 136)


def test_inner_long(wg, device):
    run_inner(wg, device, [5000, 3], 264, 392)
    run_inner(wg, device, [5000, 3], 263, 391, "float16")


@pytest.mark.parametrize("poison", [np.inf, np.nan])
def test_inner_rows_of_no_group_do_not_count(wg, device, poison):
    """Infinities and NaN in the rows around the groups reach no sum (a tile that
    a group's last row ends inside reads them)."""
    run_inner(wg, device, [20, 0, 75], 136, 200, first=3, after=9, poison=poison)
    run_inner(wg, device, [20, 0, 75], 135, 201, first=3, after=9, poison=poison)


@pytest.mark.parametrize("bad", [[0, 50, 20, 90], [-5, 10, 20, 90], [0, 10, 200, 90], [90, 0, 0, 0]])
def test_bad_offsets_are_clamped_and_reported(wg, device, bad):
    rng = np.random.default_rng(3)
    m, n, k = 90, 64, 72
    a, b = rng.standard_normal((m, k)), rng.standard_normal((3, n, k))
    (sa, va), (sb, vb) = up(wg, a, "bfloat16"), up(wg, b, "bfloat16")
    A, B = wg.GpuArray.from_(device, sa, "bfloat16"), wg.GpuArray.from_(device, sb, "bfloat16")
    C = wg.GpuArray.from_(device, np.ones(m * n, np.float32))
    off = wg.GpuArray.from_(device, np.array(bad, np.int32))
    wg._native.check(wg._native.lib.wg_gemm_grouped_dev(
        device.handle, 1, 0, 1, 3, m, n, k, 1.0, A.ptr, k, B.ptr, k, n * k, off.ptr, 0.0, C.ptr, n, None))
    with pytest.raises(wg._native.NativeError, match="offsets") as e:
        device.check()
    assert e.value.status == wg._native.WG_ERR_INVALID_ARGUMENT
    device.check()  # reported once
    want, mag = gc.rows_form(va, vb, True, bad, 1.0, 0.0, np.ones((m, n)))
    gc.assert_close(C.read().astype(np.float64).reshape(m, n), want, mag, k, 0.0, want, "float32")
    for x in (A, B, C, off):
        x.destroy()


def test_nan_and_infinity_stay_in_their_rows(wg, device):
    rng = np.random.default_rng(4)
    m, n, k = 70, 64, 72
    a = rng.standard_normal((m, k)).astype(np.float32)
    a[3, 5], a[64, 0], a[33, 71] = np.nan, np.inf, -np.inf
    A = wg.GpuArray.from_(device, a, "bfloat16")
    B = wg.GpuArray.from_(device, rng.uniform(0.5, 1, (2, n, k)).astype(np.float32), "bfloat16")
    C = wg.GpuArray.empty(device, m * n, "float32")
    off = wg.GpuArray.from_(device, np.array([0, 40, 70], np.int32))
    wg.gemmGrouped(device, T, 2, m, n, k, 1.0, A, k, B, k, n * k, off, 0.0, C, n)
    c = C.read().reshape(m, n)
    assert np.isnan(c[3]).all() and (c[64] == np.inf).all() and (c[33] == -np.inf).all()
    assert np.isfinite(np.delete(c, [3, 33, 64], 0)).all()
    for x in (A, B, C, off):
        x.destroy()


def test_results_do_not_depend_on_the_run(wg, device):
    a = run_rows(wg, device, T, [300, 0, 257, 1], 520, 1000)
    b = run_rows(wg, device, T, [300, 0, 257, 1], 520, 1000)
    assert np.array_equal(a, b)
