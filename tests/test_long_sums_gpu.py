"""Long contractions: what an accumulator of the tensor cores loses by truncating must stay
small against the rounding of the result, whatever the contraction's length."""
from __future__ import annotations

import numpy as np
import pytest

import grouped_check as gc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
T, N = "transpose", "no-transpose"
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
# A truncation keeps the sign of every error, and on data of one sign they all add up. A
# 16-bit result is a sum in 32 bits, rounded once: that sum may be off by an eighth of the
# type's half step for all truncations, and by a few roundings in 32 bits.
SHARE = 1 / 8
FEW = 2.0 ** -18


@pytest.fixture(scope="module")
def dev(wg):
    d = wg.init()
    d.set_stream(0)
    yield d
    d.set_stream(None)


def positive(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.rand(shape, generator=g, device="cuda") + 0.5).to(dtype)


def product64(a, b):
    """a b^T in 64 bits, in pieces of the contraction."""
    out = torch.zeros((a.shape[0], b.shape[0]), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 25) // max(a.shape[0], b.shape[0]))
    for i in range(0, a.shape[1], step):
        out += a[:, i:i + step].double() @ b[:, i:i + step].double().t()
    return out


def check(got, want, ctype):
    """Rounding to the type is monotone: a sum within want * (1 -+ eps) rounds to a value between the
    rounded ends of that interval."""
    eps = gc.HALF_STEP[ctype] * SHARE + FEW
    low, high = ((want * (1 + s * eps)).to(TYPES[ctype]) for s in (-1, 1))  # (want > 0)
    assert ((low <= got) & (got <= high)).all(), ((got.double() - want) / want).aminmax()


LENGTHS = [8192, 8208, 70000, 1 << 20]


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("trans", [T, N])
@pytest.mark.parametrize("k", LENGTHS)
def test_rows(wg, dev, ctype, trans, k):
    """A row for each of many groups, one matrix for all: enough tiles that none's contraction is
    split over CTAs (which drain at any length)."""
    groups, n = 256, 64
    a, b = positive((groups, k), TYPES[ctype], k), positive((n, k), TYPES[ctype], k + 1)
    alpha = 64.0 / k
    w = b if trans == T else b.t().contiguous()
    off = torch.arange(groups + 1, dtype=torch.int32, device="cuda")
    c = torch.zeros((groups, n), dtype=TYPES[ctype], device="cuda")
    wg.gemmGrouped(dev, trans, groups, groups, n, k, alpha, a, k, w, w.shape[1], 0, off, 0.0, c, n)
    dev.check()
    check(c, alpha * product64(a, b), ctype)


@pytest.mark.parametrize("ctype", TYPES)
@pytest.mark.parametrize("k", LENGTHS)
@pytest.mark.parametrize("m,n,groups", [(64, 64, 256), (130, 72, 200), (512, 520, 60)])
def test_inner(wg, dev, ctype, k, m, n, groups):
    """Two of many groups hold the rows: ragged ones of three quarters and a quarter of them."""
    if k == 1 << 20 and m > 64:
        k = 1 << 18
    a, b = positive((k, m), TYPES[ctype], k), positive((k, n), TYPES[ctype], k + 1)
    cut = k * 3 // 4 + 5
    ends = [0] * 3 + [cut] * (groups - 6) + [k] * 4
    off = torch.tensor(ends, dtype=torch.int32, device="cuda")
    alpha = 64.0 / k
    c = torch.full((groups, m, n), 7.0, dtype=TYPES[ctype], device="cuda")
    wg.gemmGroupedInner(dev, groups, m, n, k, alpha, a, m, b, n, off, 0.0, c, n, m * n)
    dev.check()
    seen = [g for g in range(groups) if ends[g] < ends[g + 1]]
    assert len(seen) == 2
    for g in seen:
        r = slice(ends[g], ends[g + 1])
        check(c[g], alpha * product64(a[r].t(), b[r].t()), ctype)
    rest = torch.ones(groups, dtype=torch.bool, device="cuda")
    rest[seen] = False
    assert (c[rest] == 0).all()


def heavy(rows, k, seed):
    """Positive values over many powers of two: their sums in 32 bits are not exact."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty((rows, k), device="cuda")
    for i in range(rows):
        x[i] = torch.exp(2.0 * torch.randn(k, generator=g, device="cuda"))
    return x


def quantized(wg, dev, x, groups=0, off=None):
    """x in MXFP4, and its values in place of x."""
    rows, k = x.shape
    q = wg.GpuMxMatrix.empty(dev, rows, k, groups=groups)
    wg.mxQuantize(dev, N, rows, k, x, k, q, offsets=off)
    wg.mxDequantize(dev, q, x, k, offsets=off)
    return q


@pytest.mark.parametrize("ctype,k", [("float16", 65536), ("float16", 65824), ("float16", 1 << 22), ("bfloat16", 1 << 19),
                                     ("bfloat16", (1 << 19) + 32), ("bfloat16", 1 << 24)])
def test_mx(wg, dev, ctype, k):
    m = 40
    x = heavy(m, k, 3)
    q = quantized(wg, dev, x)
    want = product64(x, x)
    alpha = 2.0 ** np.floor(np.log2(64.0 / want.max().item()))
    c = torch.zeros((m, m), dtype=TYPES[ctype], device="cuda")
    wg.mxGemm(dev, m, m, k, alpha, q, q, 0.0, c, m)
    dev.check()
    check(c.diagonal(), alpha * want.diagonal(), ctype)  # the largest sums, and far from fp16's subnormals
    q.destroy()


def test_mx_grouped(wg, dev):
    """The same, of rows grouped by expert."""
    m, k = 40, 1 << 22
    x = heavy(m, k, 4)
    off = torch.tensor([0, 0, m - 3, m], dtype=torch.int32, device="cuda")
    a = quantized(wg, dev, x, 3, off)
    w, b = wg.GpuMxMatrix.empty(dev, m, k), wg.GpuMxMatrix.empty(dev, m, k, batch=3)
    wg.mxQuantize(dev, N, m, k, x, k, w)  # (x holds values of the format by now)
    b.codes.write(np.tile(w.codes.read(), 3)), b.scales.write(np.tile(w.scales.read(), 3))
    want = product64(x, x)
    alpha = 2.0 ** np.floor(np.log2(64.0 / want.max().item()))
    c = torch.zeros((m, m), dtype=torch.float16, device="cuda")
    wg.mxGemmGrouped(dev, 3, m, m, k, alpha, a, b, off, 0.0, c, m)
    dev.check()
    check(c.diagonal(), alpha * want.diagonal(), "float16")
    for q in (a, b, w):
        q.destroy()


# ---- results in 32 bits: drained segments -------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans", [T, N])
def test_rows_in_32_bits(wg, dev, dtype, trans):
    """A segment is 512 rows, 32 MMAs of at most 4 additions, each off by at most 2^-23 of the
    segment's partial sums (of one sign in a segment but for its beginning: at most 2/3 of its sum on
    average over it), and 2^8 segments' sums rounded to nearest: together below 1.1e-5 of the
    result's norm. One accumulator for all would be off by 1.5e-4."""
    groups, n, k = 256, 64, 1 << 17
    g = torch.Generator(device="cuda").manual_seed(5)
    a, b = (torch.randn((r, k), generator=g, device="cuda").to(TYPES[dtype]) for r in (groups, n))
    w = b if trans == T else b.t().contiguous()
    off = torch.arange(groups + 1, dtype=torch.int32, device="cuda")
    c = torch.zeros((groups, n), device="cuda")
    wg.gemmGrouped(dev, trans, groups, groups, n, k, 1.0, a, k, w, w.shape[1], 0, off, 0.0, c, n)
    want = product64(a, b)
    assert (c.double() - want).norm() <= 1.1e-5 * want.norm()


@pytest.mark.parametrize("m", [40, 300])
def test_mx_in_32_bits(wg, dev, m):
    """A segment is 4096 rows, 64 MMAs, each off by at most 2^-23 of the segment's sum; 2^7
    segments' sums are rounded to nearest, each by at most 2^-24: below 1.6e-5. One
    accumulator for all would be off by 9e-5."""
    k = 1 << 19
    x = heavy(m, k, 6)
    q = quantized(wg, dev, x)
    c = torch.zeros((m, m), device="cuda")
    wg.mxGemm(dev, m, m, k, 1.0, q, q, 0.0, c, m)
    want = product64(x, x)
    assert (c.double() - want).norm() <= 1.6e-5 * want.norm()
    q.destroy()


# ---- the longest contractions a call takes ---------------------------------------------------
# (a wait for one accumulator's whole contraction would pass the kernels' time limit of 4e9 clocks
# here: 2^25 k-blocks take 230 clocks each)


def needs(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of free device memory")


@pytest.mark.parametrize("groups", [1, 200], ids=["split", "whole"])
def test_as_many_contraction_rows_as_a_call_takes(wg, dev, groups):
    """One group has them all, in a call that splits its contraction and in one that does not."""
    needs(72)
    k, m, n = (1 << 31) - 1025, 8, 8
    a, b = (torch.zeros((k, s), dtype=torch.bfloat16, device="cuda") for s in (m, n))
    want = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    for i, r in enumerate((slice(0, 300), slice(1 << 30, (1 << 30) + 500), slice(k - 77, k))):
        for x in (a, b):
            x[r] = positive((r.stop - r.start, m), torch.bfloat16, 10 + i)
        want += a[r].double().t() @ b[r].double()
    off = torch.full((groups + 1,), k, dtype=torch.int32, device="cuda")
    off[: groups // 2 + 1] = 0
    c = torch.full((groups, m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    wg.gemmGroupedInner(dev, groups, m, n, k, 2.0 ** -4, a, m, b, n, off, 0.0, c, n, m * n)
    dev.check()
    check(c[groups // 2], want / 16, "bfloat16")
    c[groups // 2] = 0
    assert (c == 0).all()
    del a, b
    torch.cuda.empty_cache()


def test_a_ragged_group_behind_a_very_long_one(wg, dev):
    """Two tiles of one CTA, both with rows past the last whole 16: the second's wait for its last rows
    takes as long as the first's contraction."""
    needs(72)
    first, second, m, n = (3 << 29) + 5, (1 << 26) + 7, 8, 8
    groups, other = 200, torch.cuda.get_device_properties(0).multi_processor_count
    k = first + second
    a, b = (torch.zeros((k, s), dtype=torch.bfloat16, device="cuda") for s in (m, n))
    wants = []
    for i, ends in enumerate(((0, first), (first, k))):
        spots = slice(ends[0], ends[0] + 300), slice(ends[1] - 77, ends[1])
        for x in (a, b):
            for r in spots:
                x[r] = positive((r.stop - r.start, m), torch.bfloat16, 30 + i)
        wants.append(sum(a[r].double().t() @ b[r].double() for r in spots))
    off = torch.full((groups + 1,), first, dtype=torch.int32, device="cuda")
    off[0], off[other + 1:] = 0, k
    c = torch.full((groups, m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    wg.gemmGroupedInner(dev, groups, m, n, k, 2.0 ** -4, a, m, b, n, off, 0.0, c, n, m * n)
    dev.check()
    for g, want in zip((0, other), wants):
        check(c[g], want / 16, "bfloat16")
        c[g] = 0
    assert (c == 0).all()
    del a, b
    torch.cuda.empty_cache()


def test_as_many_columns_as_an_mx_call_takes(wg, dev):
    needs(72)
    k, m = (1 << 31) - 1025, 8
    x = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    spots = (slice(0, 300), slice(1 << 30, (1 << 30) + 512), slice(k - 77, k))
    for i, r in enumerate(spots):
        x[:, r] = positive((m, r.stop - r.start), torch.bfloat16, 20 + i)
    q = wg.GpuMxMatrix.empty(dev, m, k)
    wg.mxQuantize(dev, N, m, k, x, k, q)
    wg.mxDequantize(dev, q, x, k)
    c = torch.zeros((m, m), dtype=torch.bfloat16, device="cuda")
    wg.mxGemm(dev, m, m, k, 2.0 ** -4, q, q, 0.0, c, m)
    dev.check()
    want = sum(x[:, r].double() @ x[:, r].double().t() for r in spots)
    check(c, want / 16, "bfloat16")
    q.destroy()
    del x
    torch.cuda.empty_cache()
