"""Whose memory a GpuMxMatrix is (CPU: the library's buffers are stood in for)."""
from __future__ import annotations

import pytest

from test_grouped_cpu import N, Tensor, at, dev  # noqa: F401


class Buffers:
    """wg_buffer_* over host memory; everything else is the library's."""

    def __init__(self, real):
        self.real, self.next, self.live = real, 1 << 40, set()

    def __getattr__(self, name):
        return getattr(self.real, name)

    def wg_buffer_alloc(self, device, nbytes, ref):
        self.next += 1 << 32
        self.live.add(self.next)
        ref._obj.value = self.next
        return 0

    def wg_buffer_device_ptr(self, b, ref):
        ref._obj.value = b.value
        return 0

    def wg_buffer_free(self, b):
        self.live.remove(b.value)
        return 0


@pytest.fixture()
def buffers(wg, monkeypatch):
    b = Buffers(wg._native.lib)
    monkeypatch.setattr(wg._native, "lib", b)
    return b


def test_destroy_frees_what_empty_made(wg, dev, buffers):
    q = wg.GpuMxMatrix.empty(dev, 40, 50)
    assert len(buffers.live) == 2
    q.destroy()
    assert not buffers.live
    q.destroy()  # once more is nothing


@pytest.mark.parametrize("how", ["wrap", "checked", "class"])
def test_destroy_leaves_the_callers_arrays(wg, dev, buffers, monkeypatch, how):
    codes = wg.GpuArray.empty(dev, wg.mxCodesSize(40, 50), "uint8")
    scales = wg.GpuArray.empty(dev, wg.mxScalesSize(40, 50), "uint8")
    if how == "checked":  # the same through the Python checks
        class Never:
            def __getattr__(self, name):
                return lambda *a: None

        monkeypatch.setattr(wg._native, "_fast", Never())
    q = wg.GpuMxMatrix(dev, codes, scales, 40, 50, 1, 0) if how == "class" else wg.GpuMxMatrix.wrap(dev, codes, scales, 40, 50)
    again = wg.GpuMxMatrix.wrap(dev, codes, scales, 40, 50)
    q.destroy()
    assert len(buffers.live) == 2 and codes.ptr and scales.ptr and codes.length == wg.mxCodesSize(40, 50)
    assert again._codes == codes.ptr
    with pytest.raises(wg.Error):  # the destroyed one takes no part any more
        wg.mxQuantize(dev, N, 40, 50, Tensor(2000, "bfloat16", at(0)), 50, q)
    codes.destroy(), scales.destroy()
    assert not buffers.live
