"""Which stream a handle's work is ordered on, as other libraries name streams: the
number 0 is their default stream, and the documented way to take torch's holds on it."""
from __future__ import annotations

import ctypes as ct
import os
import re

import numpy as np
import pytest

import grouped_check as gc
from conftest import ROOT

LEGACY = 1  # cudaStreamLegacy


@pytest.fixture()
def stand_in(wg):
    """A device over zeroed memory: its own stream is the handle 0."""
    block = (ct.c_char * 65536)()
    yield wg.Device(ct.cast(block, ct.c_void_p), 0, False, {}, "stand-in")


def test_the_number_zero_is_the_default_stream(stand_in):
    """torch.cuda.default_stream().cuda_stream is 0, and so is cudaStream_t 0 everywhere."""
    for stream, want in ((0, LEGACY), (np.int64(0), LEGACY), (LEGACY, LEGACY), (2, 2), (1 << 40, 1 << 40), (None, 0)):
        stand_in.set_stream(stream)
        assert stand_in.stream() == want, stream


def layer_example():
    """The layer's step in the integration notes, as a user copies it."""
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    code = [c for c in re.findall(r"```python\n(.*?)```", text, re.S) if "gemmGroupedInner" in c]
    assert len(code) == 1
    return code[0]


@pytest.mark.gpu
@pytest.mark.parametrize("side", [False, True], ids=["default", "side"])
@pytest.mark.parametrize("n,k", [(256, 512), (131, 201)])
def test_the_documented_step_is_ordered_with_torch(wg, side, n, k):
    """Word for word, with torch work that writes the operands still running before it and
    torch work that reads the results queued behind it."""
    torch = pytest.importorskip("torch")
    code = layer_example()
    sizes = [100, 0, 300]
    G, m = 3, sum(sizes)
    ends = np.concatenate([[0], np.cumsum(sizes)])
    stream = torch.cuda.Stream() if side else torch.cuda.default_stream()
    g = torch.Generator(device="cuda").manual_seed(n)
    x, w, dy = (torch.randn(s, generator=g, device="cuda").bfloat16() for s in ((m, k), (G, n, k), (m, n)))
    off = torch.tensor(ends, dtype=torch.int32, device="cuda")
    names = dict(wg=wg, torch=torch, G=G, m=m, n=n, k=k, X=torch.zeros_like(x), W=torch.zeros_like(w),
                 dY=torch.zeros_like(dy), offsets=torch.zeros_like(off),
                 Y=torch.zeros((m, n), dtype=torch.bfloat16, device="cuda"),
                 dX=torch.zeros((m, k), dtype=torch.bfloat16, device="cuda"), dW=torch.ones((G, n, k), device="cuda"))
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(stream):
            for _ in range(20):
                big = big @ big * 1e-3  # tens of milliseconds in front of the operands
            for name, value in (("X", x), ("W", w), ("dY", dy), ("offsets", off)):
                names[name].copy_(value)
            exec(code, names)
            got = [names[r].clone() for r in ("Y", "dX", "dW")]
            for r in ("Y", "dX", "dW"):
                names[r].zero_()
        torch.cuda.synchronize()
        names["dev"].check()
    finally:
        wg.init().set_stream(None)
    xs, ws, ds = (t.double().cpu().numpy() for t in (x, w, dy))
    want, mag = gc.rows_form(xs, ws, True, ends, 1.0, 0.0, np.zeros((m, n)))
    gc.assert_close(got[0].double().cpu().numpy(), want, mag, k, 0.0, np.zeros(1), "bfloat16", "Y")
    want, mag = gc.rows_form(ds, ws, False, ends, 1.0, 0.0, np.zeros((m, k)))
    gc.assert_close(got[1].double().cpu().numpy(), want, mag, n, 0.0, np.zeros(1), "bfloat16", "dX")
    one = np.ones((G, n, k))
    want, mag = gc.inner_form(ds, xs, ends, 1.0, 1.0, one)
    gc.assert_close(got[2].double().cpu().numpy(), want, mag, m, 1.0, one, "float32", "dW")


@pytest.mark.gpu
def test_the_other_routines_on_the_default_stream(wg):
    """Host-array and resident calls give the same bits as on the handle's own stream."""
    dev = wg.init()

    def results():
        out = []
        for m, n, k in ((70, 50, 90), (640, 1100, 700), (2304, 2304, 2304)):
            a, b = wg.randomNormalFloat32Array(m * k, 1), wg.randomNormalFloat32Array(k * n, 2)
            c = np.zeros(m * n, np.float32)
            out.append(wg.sgemm(dev, "no-transpose", "no-transpose", m, n, k, 1.5, a, k, b, n, 0.0, c, n)["C"])
            ga, gb = (wg.GpuMatrix.from_(dev, v, r, s) for v, r, s in ((a, m, k), (b, k, n)))
            gcm = wg.GpuMatrix.from_(dev, np.zeros(m * n, np.float32), m, n)
            wg.sgemm(dev, "no-transpose", "no-transpose", m, n, k, 1.5, ga, k, gb, n, 0.0, gcm, n)
            out.append(np.asarray(gcm.read()).copy())
            for x in (ga, gb, gcm):
                x.destroy()
        n = 300
        tri = np.tril(wg.randomNormalFloat32Array(n * n, 3).reshape(n, n)) + 20 * np.eye(n, dtype=np.float32)
        tri = tri.astype(np.float32).reshape(-1)
        rhs, x, y = wg.randomNormalFloat32Array(n * 40, 4), wg.randomNormalFloat32Array(n, 5), np.zeros(n, np.float32)
        out.append(wg.strsm(dev, "left", "lower", "no-transpose", "non-unit", n, 40, 1.0, tri, n, rhs, 40)["B"])
        out.append(wg.sgemv(dev, "no-transpose", n, n, 1.0, tri, n, x, 1, 0.0, y, 1)["y"])
        return out

    try:
        dev.set_stream(None)
        own = results()
        dev.set_stream(0)
        default = results()
    finally:
        dev.set_stream(None)
    for i, (a, b) in enumerate(zip(own, default)):
        assert np.abs(a).max() > 0 and np.array_equal(a, b), i
