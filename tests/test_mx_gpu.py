"""MXFP4 quantisation and products on the GPU against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import grouped_check as gc
import mx_check as mc
from test_grouped_gpu import up, values

pytestmark = pytest.mark.gpu

T, N = "transpose", "no-transpose"


def data(rng, rows, cols):
    """Values over many magnitudes, with exact ties, zeros and whole blocks of zeros."""
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 12, (rows, cols)).astype(float))
    x[rng.random((rows, cols)) < 0.1] = 0
    t = rng.random((rows, cols)) < 0.3
    x[t] = (rng.integers(-16, 17, (rows, cols)) / 4.0)[t]
    for r in range(0, rows, 3):
        x[r, 32:64] = 0
        x[r, :32] *= 2.0 ** rng.integers(-8, 8)
    return x.astype(np.float32)


def quantized(wg, device, x, dtype="float32", trans=N, ld=None, offsets=None, groups=0):
    """(GpuMxMatrix, values given) of quantising the matrix whose op() is x."""
    rows, cols = x.shape
    s = x.T if trans == T else x
    ld = ld or s.shape[1]
    full = np.full((s.shape[0], ld), np.nan, np.float32)
    full[:, : s.shape[1]] = s
    st, va = up(wg, full.reshape(-1), dtype)
    X = wg.GpuArray.from_(device, st, dtype)
    q = wg.GpuMxMatrix.empty(device, rows, cols, groups=groups)
    q.codes.write(np.full(q.codes.length, 0xEE, np.uint8))
    q.scales.write(np.full(q.scales.length, 0xEE, np.uint8))
    off = None if offsets is None else wg.GpuArray.from_(device, np.asarray(offsets, np.int32))
    wg.mxQuantize(device, trans, rows, cols, X, ld, q, offsets=off)
    device.check()
    X.destroy()
    va = va.reshape(s.shape[0], ld)[:, : s.shape[1]]
    return q, (va.T if trans == T else va)


@pytest.mark.parametrize("trans", [N, T])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 33), (128, 128), (129, 127), (40, 300), (257, 64), (5, 1023),
                                       (300, 8), (64, 512)])
def test_quantize(wg, device, trans, dtype, rows, cols):
    rng = np.random.default_rng(rows * 1000 + cols)
    x = data(rng, rows, cols)
    if dtype == "float16":
        x = np.clip(x, -60000, 60000)
    for ld in (None, (rows if trans == T else cols) + 3):
        q, x64 = quantized(wg, device, x, dtype, trans, ld)
        code, scale = mc.quantize(x64)
        assert np.array_equal(q.codes.read().reshape(rows, -1), mc.pack_codes(code))
        assert np.array_equal(q.scales.read(), mc.tile_scales(scale))
        want = mc.values(code, scale, cols)
        assert np.array_equal(wg.mxDecode(q.codes.read(), q.scales.read(), rows, cols), want)
        out = wg.GpuArray.from_(device, np.full(rows * (cols + 1), 7, np.float32))
        wg.mxDequantize(device, q, out, cols + 1)
        got = out.read().reshape(rows, cols + 1)
        assert np.array_equal(got[:, :cols], want) and (got[:, cols] == 7).all()
        out.destroy()
        q.destroy()


def test_quantize_extremes(wg, device):
    """Subnormals, the largest values, infinities and NaN (whose block is NaN), signed zeros."""
    x = np.zeros((4, 160), np.float32)
    x[0, :32] = np.float32(1e-45)
    x[0, 32:64] = np.linspace(-1.2e-38, 1.2e-38, 32)
    x[0, 64:96] = 3.4028235e38
    x[0, 96:128] = np.float32(2.0 ** 127) * np.linspace(0, 1, 32).astype(np.float32)
    x[1, 5], x[1, 40], x[1, 70] = np.nan, np.inf, -np.inf
    x[1, 96:128] = -0.0
    x[2] = np.tile(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7], np.float32), 20)
    x[2, ::2] *= -1
    x[3, :32] = 2.0 ** -126
    q, x64 = quantized(wg, device, x)
    code, scale = mc.quantize(x64)
    ok = np.repeat(scale != 255, 32, 1)
    got = q.codes.read().reshape(4, -1)
    pairs = np.stack([got & 15, got >> 4], -1).reshape(4, -1)
    assert np.array_equal(pairs[ok], code[ok])
    assert np.array_equal(q.scales.read(), mc.tile_scales(scale))
    out = wg.GpuArray.empty(device, 4 * 160, "float32")
    wg.mxDequantize(device, q, out, 160)
    got = out.read().reshape(4, 160).astype(np.float64)
    assert np.array_equal(got, mc.values(code, scale, 160), equal_nan=True)
    for d in ("bfloat16", "float16"):
        o = wg.GpuArray.empty(device, 4 * 160, d)
        wg.mxDequantize(device, q, o, 160)
        with np.errstate(over="ignore"):
            _, want = up(wg, mc.values(code, scale, 160).astype(np.float32), d)
        assert np.array_equal(values(wg, o).reshape(4, 160), want, equal_nan=True)
        o.destroy()
    out.destroy()
    q.destroy()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols", [(31, 1000), (333, 777), (1000, 1000), (7205, 2056)])
def test_quantize_there_and_back(wg, device, dtype, rows, cols):
    """Quarters of tile pairs and whole ones, rows of whole 16-byte units and others, in both directions."""
    rng = np.random.default_rng(rows + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-8, 8, (rows, 1)))).astype(np.float32)
    for pad in (0, 8, 3):
        q, x64 = quantized(wg, device, x, dtype, ld=cols + pad)
        if pad == 0:
            code, scale = mc.quantize(x64)
            want_codes, want_scales = mc.pack_codes(code), mc.tile_scales(scale)
            want = mc.values(code, scale, cols)
            assert (want == want.astype(np.float32)).all()
        assert np.array_equal(q.codes.read().reshape(rows, -1), want_codes)
        assert np.array_equal(q.scales.read(), want_scales)
        blank = up(wg, np.full(rows * (cols + pad), 7, np.float32), dtype)[0]
        out = wg.GpuArray.from_(device, blank, dtype)
        wg.mxDequantize(device, q, out, cols + pad)
        got = values(wg, out).reshape(rows, cols + pad)
        # (4-bit elements times a power of two in range: exact in every type)
        assert np.array_equal(got[:, :cols], want) and (got[:, cols:] == 7).all()
        out.destroy()
        q.destroy()


@pytest.mark.parametrize("sizes,first,after", [([5, 0, 130, 1], 0, 0), ([128, 128], 0, 3), ([0, 300], 4, 2), ([0], 2, 0)])
def test_quantize_grouped_rows(wg, device, sizes, first, after):
    rng = np.random.default_rng(9)
    cuts = first + np.concatenate([[0], np.cumsum(sizes)])
    rows, cols = int(cuts[-1]) + after, 200
    x = data(rng, rows, cols)
    q, x64 = quantized(wg, device, x, offsets=cuts, groups=len(sizes))
    code, scale = mc.quantize(x64)
    got, want = q.codes.read().reshape(rows, -1), mc.pack_codes(code)
    inside = slice(int(cuts[0]), int(cuts[-1]))
    assert np.array_equal(got[inside], want[inside])
    assert (np.delete(got, np.r_[inside], 0) == 0xEE).all()  # rows of no group
    tiles = mc.tile_scales(scale, cuts)
    s = q.scales.read()
    assert np.array_equal(s[: tiles.size], tiles) and (s[tiles.size:] == 0xEE).all()
    out = wg.GpuArray.from_(device, np.full(rows * cols, 7, np.float32))
    off = wg.GpuArray.from_(device, cuts.astype(np.int32))
    wg.mxDequantize(device, q, out, cols, offsets=off)
    o = out.read().reshape(rows, cols)
    assert np.array_equal(o[inside], mc.values(code, scale, cols)[inside])
    assert (np.delete(o, np.r_[inside], 0) == 7).all()
    for y in (out, off, q):
        y.destroy()


def test_quantize_batch(wg, device):
    rng = np.random.default_rng(11)
    batch, rows, cols = 3, 130, 72
    for trans in (N, T):
        sr, sc = (cols, rows) if trans == T else (rows, cols)
        stride = sr * sc + 5
        x = np.full(batch * stride, np.nan, np.float32)
        mats = [data(rng, rows, cols) for _ in range(batch)]
        for i, m in enumerate(mats):
            x[i * stride: i * stride + sr * sc] = (m.T if trans == T else m).reshape(-1)
        X = wg.GpuArray.from_(device, x)
        q = wg.GpuMxMatrix.empty(device, rows, cols, batch=batch)
        wg.mxQuantize(device, trans, rows, cols, X, sc, q, strideX=stride)
        codes, scales = q.codes.read().reshape(batch, rows, -1), q.scales.read().reshape(batch, -1)
        out = wg.GpuArray.empty(device, batch * rows * cols, "float32")
        wg.mxDequantize(device, q, out, cols)
        o = out.read().reshape(batch, rows, cols)
        for i, m in enumerate(mats):
            code, scale = mc.quantize(m)
            assert np.array_equal(codes[i], mc.pack_codes(code))
            assert np.array_equal(scales[i], mc.tile_scales(scale))
            assert np.array_equal(o[i], mc.values(code, scale, cols))
        for y in (X, q, out):
            y.destroy()


def operand(rng, rows, cols):
    return (rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((1, cols)))).astype(np.float32)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 64), (16, 128, 256), (33, 40, 100), (128, 128, 128), (130, 257, 300),
                                   (200, 130, 512), (300, 200, 1000), (513, 260, 2048), (5, 1000, 96), (260, 64, 65)])
@pytest.mark.parametrize("ctype", ["float32", "bfloat16"])
def test_gemm(wg, device, m, n, k, ctype):
    rng = np.random.default_rng(m + n + k)
    a, va = quantized(wg, device, operand(rng, m, k))
    b, vb = quantized(wg, device, operand(rng, n, k))
    va, vb = mc.values(*mc.quantize(va), k), mc.values(*mc.quantize(vb), k)
    ldc = n + (n & 3)
    c0, vc = up(wg, np.full(m * ldc, np.nan, np.float32), ctype)
    C = wg.GpuArray.from_(device, c0, ctype)
    wg.mxGemm(device, m, n, k, 1.0, a, b, 0.0, C, ldc)
    device.check()
    got = values(wg, C).reshape(m, ldc)
    gc.assert_close(got[:, :n], va @ vb.T, np.abs(va) @ np.abs(vb).T, k, 0.0, np.zeros((m, n)), ctype, "C")
    assert np.isnan(got[:, n:]).all()
    for x in (a, b, C):
        x.destroy()


@pytest.mark.parametrize("m,n,k", [(2560, 2048, 128), (2570, 2050, 330), (1300, 4100, 1024), (700, 9700, 200),
                                   (150, 20000, 96)])
@pytest.mark.parametrize("ctype", ["float32", "bfloat16"])
def test_gemm_pairs(wg, device, m, n, k, ctype):
    test_gemm(wg, device, m, n, k, ctype)


@pytest.mark.parametrize("m,n,k", [(1, 200, 4096), (20, 1000, 8192), (33, 260, 3000), (64, 520, 5000), (100, 136, 2048),
                                   (5, 8192, 1024), (40, 8192, 1100)])
@pytest.mark.parametrize("ctype", ["float32", "bfloat16"])
def test_gemm_few_rows(wg, device, m, n, k, ctype):
    """Narrow tiles, and contractions split over several CTAs."""
    test_gemm(wg, device, m, n, k, ctype)


@pytest.mark.parametrize("m,n,k", [(64, 130, 9000), (2570, 2050, 4500)])
def test_gemm_long(wg, device, m, n, k):
    test_gemm(wg, device, m, n, k, "float32")


@pytest.mark.parametrize("ctype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("alpha,beta", [(0.5, 1.0), (-2.0, 0.25), (0.0, 0.0), (0.0, -1.5), (0.0, 1.0)])
def test_gemm_scalars(wg, device, ctype, alpha, beta):
    rng = np.random.default_rng(5)
    m, n, k = 140, 136, 200
    a, va = quantized(wg, device, rng.standard_normal((m, k)).astype(np.float32))
    b, vb = quantized(wg, device, rng.standard_normal((n, k)).astype(np.float32))
    va, vb = mc.values(*mc.quantize(va), k), mc.values(*mc.quantize(vb), k)
    c0, vc = up(wg, rng.standard_normal(m * n).astype(np.float32), ctype)
    vc = vc.reshape(m, n)
    C = wg.GpuArray.from_(device, c0, ctype)
    wg.mxGemm(device, m, n, k, alpha, a, b, beta, C, n)
    want = alpha * (va @ vb.T) + beta * vc
    mag = abs(alpha) * (np.abs(va) @ np.abs(vb).T)
    gc.assert_close(values(wg, C).reshape(m, n), want, mag, k, beta, vc, ctype, "C")
    for x in (a, b, C):
        x.destroy()


def test_gemm_nan_blocks(wg, device):
    """A block that is not a number makes its row of the product (and its column) NaN, no other."""
    rng = np.random.default_rng(6)
    m, n, k = 70, 136, 300
    x, w = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((n, k)).astype(np.float32)
    x[3, 299], x[64, 0], w[100, 64] = np.nan, np.inf, -np.inf
    a, _ = quantized(wg, device, x)
    b, _ = quantized(wg, device, w)
    C = wg.GpuArray.empty(device, m * n, "float32")
    wg.mxGemm(device, m, n, k, 1.0, a, b, 0.0, C, n)
    c = C.read().reshape(m, n)
    bad = np.zeros((m, n), bool)
    bad[[3, 64]] = True
    bad[:, 100] = True
    assert np.array_equal(np.isnan(c), bad)
    for y in (a, b, C):
        y.destroy()


@pytest.mark.parametrize("sizes,first,after", [([1], 0, 0), ([5, 0, 11], 0, 4), ([0, 130, 1, 0], 2, 0), ([300, 257], 0, 0),
                                               ([64] * 9, 0, 1), ([1] * 40, 0, 0), ([0, 0], 3, 3), ([140, 0, 129, 256], 1, 0)])
@pytest.mark.parametrize("n,k", [(128, 64), (200, 300), (40, 1000)])
def test_gemm_grouped(wg, device, sizes, first, after, n, k):
    rng = np.random.default_rng(sum(sizes) + n)
    groups = len(sizes)
    cuts = first + np.concatenate([[0], np.cumsum(sizes)])
    m = int(cuts[-1]) + after
    a, va = quantized(wg, device, operand(rng, m, k), offsets=cuts, groups=groups)
    w = np.stack([operand(rng, n, k) for _ in range(groups)])
    W = wg.GpuArray.from_(device, w)
    b = wg.GpuMxMatrix.empty(device, n, k, batch=groups)
    wg.mxQuantize(device, N, n, k, W, k, b)
    va = mc.values(*mc.quantize(va), k)
    vb = np.stack([mc.values(*mc.quantize(x), k) for x in w])
    c0 = rng.standard_normal((m, n)).astype(np.float32)
    C = wg.GpuArray.from_(device, c0)
    off = wg.GpuArray.from_(device, cuts.astype(np.int32))
    wg.mxGemmGrouped(device, groups, m, n, k, 1.0, a, b, off, 0.5, C, n)
    device.check()
    want, mag = gc.rows_form(va, vb, True, cuts, 1.0, 0.5, c0.astype(np.float64))
    gc.assert_close(values(wg, C).reshape(m, n), want, mag, k, 0.5, c0.astype(np.float64), "float32", "C")
    for x in (a, b, W, C, off):
        x.destroy()


@pytest.mark.parametrize("sizes", [[3], [40, 0, 70], [1] * 9, [17] * 12, [130, 5]], ids=lambda s: f"{len(s)}g{sum(s)}")
@pytest.mark.parametrize("n,k", [(264, 4096), (1000, 1100)])
def test_gemm_grouped_few_rows(wg, device, sizes, n, k):
    test_gemm_grouped(wg, device, sizes, 1, 2, n, k)


@pytest.mark.parametrize("n,k", [(2048, 128), (2050, 600)])
def test_gemm_grouped_pairs(wg, device, n, k):
    test_gemm_grouped(wg, device, [150, 0, 1, 290, 256, 257, 31, 140, 513, 160, 64, 130, 129, 200, 300], 1, 5, n, k)
