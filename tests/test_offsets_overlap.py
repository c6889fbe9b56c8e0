"""A call that would write over the offsets it is reading is refused: CTAs read them at different
times, and those of one cluster have to see the same ones."""
from __future__ import annotations

import pytest

from test_grouped_cpu import G, M, N, NN, K, Tensor, at, dev, grouped_args, inner_args, mx, quant_args, reached  # noqa: F401


def both(wg, fast, fn, args, text):
    """Refused by the fast path, and by the Python checks with a message."""
    assert getattr(wg._native._fast, fast)(*args) is None
    with pytest.raises(wg.Error, match=text):
        fn(*args)


# Places of `size` bytes of offsets: over a result of `n` bytes at `p`, and just outside it.
def over(p, n, size):
    return (p, p + n - 4, p - size + 4)


def beside(p, n, size):
    return (p + n, p - size)


def test_grouped(wg, dev):
    size, n = 4 * (G + 1), M * NN * 2
    for where in over(at(3), n, size):
        both(wg, "gemm_grouped", wg.gemmGrouped, grouped_args(wg, dev, offsets=Tensor(G + 1, "int32", where)),
             "C must not overlap offsets")
    for where in beside(at(3), n, size):
        reached(wg, wg.gemmGrouped, *grouped_args(wg, dev, offsets=Tensor(G + 1, "int32", where)))


def test_inner(wg, dev):
    size, n = 4 * (G + 1), G * NN * K * 4
    for where in over(at(3), n, size):
        both(wg, "gemm_grouped_inner", wg.gemmGroupedInner, inner_args(wg, dev, offsets=Tensor(G + 1, "int32", where)),
             "C must not overlap offsets")
    for where in beside(at(3), n, size):
        reached(wg, wg.gemmGroupedInner, *inner_args(wg, dev, offsets=Tensor(G + 1, "int32", where)))


@pytest.mark.parametrize("part,bytes_of", [(10, "mxCodesSize"), (11, "mxScalesSize")])
def test_quantize(wg, dev, part, bytes_of):
    n = getattr(wg, bytes_of)(40, 50, *(() if part == 10 else (1, 2)))
    for where in over(at(part), n, 12):
        both(wg, "mx_quantize", wg.mxQuantize,
             quant_args(wg, dev, out=mx(wg, dev, 40, 50, groups=2), offsets=Tensor(3, "int32", where)),
             "out must not overlap offsets")
    for where in beside(at(part), n, 12):
        reached(wg, wg.mxQuantize, *quant_args(wg, dev, out=mx(wg, dev, 40, 50, groups=2), offsets=Tensor(3, "int32", where)))


def test_dequantize(wg, dev):
    def args(where):
        return [dev, mx(wg, dev, 40, 50, groups=2), Tensor(2000, "float32", at(0)), 50, Tensor(3, "int32", where), 0]

    for where in over(at(0), 8000, 12):
        both(wg, "mx_dequantize", wg.mxDequantize, args(where), "out must not overlap offsets")
    for where in beside(at(0), 8000, 12):
        reached(wg, wg.mxDequantize, *args(where))


def test_mx_gemm_grouped(wg, dev):
    def args(where):
        return [dev, 2, 40, 30, 50, 1.0, mx(wg, dev, 40, 50, groups=2), mx(wg, dev, 30, 50, batch=2, base=12),
                Tensor(3, "int32", where), 0.0, Tensor(1200, "bfloat16", at(0)), 30]

    for where in over(at(0), 2400, 12):
        a = args(where)
        assert wg._native._fast.mx_gemm(*a) is None
        with pytest.raises(wg.Error, match="C must not overlap offsets"):
            wg.mxGemmGrouped(*a)
    for where in beside(at(0), 2400, 12):
        reached(wg, wg.mxGemmGrouped, *args(where))
