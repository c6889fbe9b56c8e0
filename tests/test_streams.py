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
