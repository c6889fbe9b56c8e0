"""The grouped and MXFP4 products as a program uses them: on another library's CUDA
tensors and streams, captured into graphs, past 32-bit offsets, and together as a
layer's training step and its serving in 4 bits."""
from __future__ import annotations

import numpy as np
import pytest

import grouped_check as gc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
T, N = "transpose", "no-transpose"
LEGACY = 1  # torch's default stream


@pytest.fixture(scope="module")
def dev(wg):
    """A device without times, ordered on torch's default stream."""
    d = wg.init()
    d.set_stream(LEGACY)
    yield d
    d.set_stream(None)


def offsets_of(sizes):
    return torch.tensor([0] + list(np.cumsum(sizes)), dtype=torch.int32, device="cuda")


def make(sizes, n, k, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = sum(sizes)
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype)
    w = (torch.randn((len(sizes), n, k), generator=g, device="cuda") * k ** -0.5).to(dtype)
    return x, w, offsets_of(sizes)


def rows64(x, w, off, trans=True):
    """(product, sum of |terms|) in 64 bits."""
    ends = off.tolist()
    n = w.shape[1] if trans else w.shape[2]
    y, mag = (torch.zeros((x.shape[0], n), dtype=torch.float64, device="cuda") for _ in range(2))
    for g in range(w.shape[0]):
        r = slice(ends[g], ends[g + 1])
        a, b = x[r].double(), w[g].double().t() if trans else w[g].double()
        y[r], mag[r] = a @ b, a.abs() @ b.abs()
    return y, mag


def check(got, want, mag, k, ctype):
    gc.assert_close(got.double().cpu().numpy(), want.cpu().numpy(), mag.cpu().numpy(), k, 0.0, np.zeros(1), ctype, "C")


def forward(wg, dev, x, w, off, y):
    g, n, k = w.shape
    wg.gemmGrouped(dev, T, g, x.shape[0], n, k, 1.0, x, k, w, k, n * k, off, 0.0, y, n)


# ---- streams, views, devices -----------------------------------------------------


def test_work_is_ordered_on_the_stream_given(wg, dev):
    x, w, off = make([700, 0, 900], 1024, 2048)
    y = torch.zeros((1600, 1024), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    try:
        dev.set_stream(s.cuda_stream)
        with torch.cuda.stream(s):
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(10):
                big = big @ big * 1e-3  # keeps the stream busy: the product must wait for what follows
            x2 = x * 2
            forward(wg, dev, x2, w, off, y)
            z = y.clone()
        s.synchronize()
    finally:
        dev.set_stream(LEGACY)
    want, mag = rows64(x2, w, off)
    check(z, want, mag, 2048, "bfloat16")


def test_strided_views(wg, dev):
    """Views with a row length of their own, and bases inside a tensor."""
    sizes, n, k = [40, 3, 90], 136, 200
    m = sum(sizes)
    big = torch.randn((m + 2, k + 24), device="cuda").to(torch.bfloat16)
    x = big[1:m + 1, 8:8 + k]
    _, w, off = make(sizes, n, k)
    out = torch.full((m, n + 8), 7.0, dtype=torch.float32, device="cuda")
    y = out[:, :n]
    wg.gemmGrouped(dev, T, 3, m, n, k, 1.0, x, k + 24, w, k, n * k, off, 0.0, y, n + 8)
    want, mag = rows64(x, w, off)
    check(y, want, mag, k, "float32")
    assert (out[:, n:] == 7).all()
    with pytest.raises(wg.Error, match="A does not have enough elements"):
        wg.gemmGrouped(dev, T, 3, m + 2, n, k, 1.0, x, k + 24, w, k, n * k, off, 0.0,
                       torch.empty((m + 2, n), device="cuda"), n)


@pytest.mark.parametrize("stride,ld", [(8, 64), (64, 64), (3, 70), (0, 64)])
@pytest.mark.parametrize("trans", [N, T])
def test_experts_whose_matrices_overlap(wg, dev, trans, stride, ld):
    """Weights that share memory (windows of one matrix, or one matrix for all) are only read."""
    sizes, n, k = [40, 0, 90, 7], 48, 64
    rows, cols = (n, k) if trans == T else (k, n)
    flat = torch.randn(3 * stride + rows * ld, device="cuda").to(torch.bfloat16)
    w = torch.stack([flat[g * stride:g * stride + rows * ld].view(rows, ld)[:, :cols] for g in range(4)])
    x, _, off = make(sizes, n, k)
    y = torch.zeros((sum(sizes), n), device="cuda")
    wg.gemmGrouped(dev, trans, 4, sum(sizes), n, k, 1.0, x, k, flat, ld, stride, off, 0.0, y, n)
    want, mag = rows64(x, w, off, trans == T)
    check(y, want, mag, k, "float32")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 5, 7])
@pytest.mark.parametrize("rows,cols", [(1, 5), (3, 40), (70, 301), (129, 520)])
def test_quantize_alignment_of_the_bases(wg, dev, dtype, shift, rows, cols):
    """A matrix anywhere in memory gives the codes of its aligned copy, and back, and its neighbours stay."""
    flat = torch.full((shift + rows * cols + 9,), float("nan"), device="cuda", dtype=dtype)
    x = flat[shift:shift + rows * cols].view(rows, cols)
    x.copy_(torch.randn(rows, cols, device="cuda"))
    pitch = -(-cols // 8) * 8
    copy = torch.zeros((rows, pitch), device="cuda", dtype=dtype)
    copy[:, :cols] = x
    for trans in (N, T):
        r, c = (cols, rows) if trans == T else (rows, cols)
        q, want = wg.GpuMxMatrix.empty(dev, r, c), wg.GpuMxMatrix.empty(dev, r, c)
        wg.mxQuantize(dev, trans, r, c, x, cols, q)
        wg.mxQuantize(dev, trans, r, c, copy, pitch, want)
        assert (q.codes.read() == want.codes.read()).all() and (q.scales.read() == want.scales.read()).all()
        out = torch.full((shift + r * c + 9,), 7.0, device="cuda", dtype=dtype)
        wg.mxDequantize(dev, q, out[shift:], c)
        back = out[shift:shift + r * c].double().cpu().numpy().reshape(r, c)
        assert (back == wg.mxDecode(q.codes.read(), q.scales.read(), r, c)).all()
        assert (out[:shift] == 7).all() and (out[shift + r * c:] == 7).all()
        q.destroy(), want.destroy()


def test_a_host_tensor_is_refused(wg, dev):
    x, w, off = make([4], 8, 8)
    with pytest.raises(wg.Error, match="A must be a GpuArray or a CUDA tensor."):
        wg.gemmGrouped(dev, T, 1, 4, 8, 8, 1.0, x.cpu(), 8, w, 8, 64, off, 0.0, torch.empty_like(x), 8)


def test_benchmark_device_reports_its_time(wg, device):
    x, w, off = make([64], 64, 64)
    y = torch.empty((64, 64), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    r = wg.gemmGrouped(device, T, 1, 64, 64, 64, 1.0, x, 64, w, 64, 4096, off, 0.0, y, 64)
    assert r["gpuTimeMs"] > 0
    q = wg.GpuMxMatrix.empty(device, 64, 64)
    assert wg.mxQuantize(device, N, 64, 64, x, 64, q)["gpuTimeMs"] > 0
    assert wg.mxDequantize(device, q, y, 64)["gpuTimeMs"] > 0
    assert wg.mxGemm(device, 64, 64, 64, 1.0, q, q, 0.0, y, 64)["gpuTimeMs"] > 0
    q.destroy()


# ---- graphs ---------------------------------------------------------------------------


def capture(dev, fn):
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    try:
        dev.set_stream(s.cuda_stream)
        with torch.cuda.graph(g, stream=s):
            fn()
    finally:
        dev.set_stream(LEGACY)
    return g


@pytest.mark.parametrize("n,k", [(256, 512), (130, 201)])
def test_captured_calls_replay_on_new_inputs(wg, dev, n, k):
    sizes = [100, 0, 257, 30]
    x, w, off = make(sizes, n, k, torch.float16)
    m = sum(sizes)
    dy = torch.randn((m, n), device="cuda").half()
    y, dx = torch.zeros((m, n), device="cuda"), torch.zeros((m, k), device="cuda")
    dw = torch.zeros((4, n, k), device="cuda")
    q, wq = wg.GpuMxMatrix.empty(dev, m, k, groups=4), wg.GpuMxMatrix.empty(dev, n, k, batch=4)
    yq = torch.zeros((m, n), device="cuda")

    def step():
        forward(wg, dev, x, w, off, y)
        wg.gemmGrouped(dev, N, 4, m, k, n, 1.0, dy, n, w, k, n * k, off, 0.0, dx, k)
        wg.gemmGroupedInner(dev, 4, n, k, m, 1.0, dy, n, x, k, off, 0.0, dw, k, n * k)
        wg.mxQuantize(dev, N, n, k, w, k, wq)
        wg.mxQuantize(dev, N, m, k, x, k, q, offsets=off)
        wg.mxGemmGrouped(dev, 4, m, n, k, 1.0, q, wq, off, 0.0, yq, n)

    g = capture(dev, step)
    for seed in (1, 2):
        x2, w2, _ = make(sizes, n, k, torch.float16, seed)
        new = offsets_of([30, 200, 100, 57] if seed == 2 else sizes)  # the groups' sizes are read at replay
        x.copy_(x2), w.copy_(w2), off.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, dx, dw, yq)]
        want, mag = rows64(x, w, off)
        check(y, want, mag, k, "float32")
        step()  # eager on the same inputs: the same bits
        torch.cuda.synchronize()
        for a, b in zip(got, (y, dx, dw, yq)):
            assert torch.equal(a, b)
    dev.check()
    q.destroy(), wq.destroy()


def test_graphs_of_unaligned_calls_share_nothing(wg, dev):
    """Two captured calls that copy their operands, replayed on two streams at once, and
    eager calls between them."""
    jobs = []
    for seed in range(2):
        x, w, off = make([300 + seed, 200], 515, 1003, torch.float16, seed)
        y = torch.zeros((x.shape[0], 515), device="cuda")
        jobs.append((x, w, off, y, capture(dev, lambda x=x, w=w, off=off, y=y: forward(wg, dev, x, w, off, y))))
    streams = [torch.cuda.Stream() for _ in jobs]
    xe, we, offe = make([77, 5], 131, 999, torch.float16, 9)
    ye = torch.zeros((82, 131), device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        for (x, w, off, y, g), s in zip(jobs, streams):
            with torch.cuda.stream(s):
                g.replay()
        forward(wg, dev, xe, we, offe, ye)
    torch.cuda.synchronize()
    for x, w, off, y, g in jobs:
        want, mag = rows64(x, w, off)
        check(y, want, mag, 1003, "float32")
    want, mag = rows64(xe, we, offe)
    check(ye, want, mag, 999, "float32")


def test_two_streams_with_unaligned_operands(wg, dev):
    """The handle moved between streams while the first one's copies are still in use."""
    s = torch.cuda.Stream()
    a, b = make([900], 513, 1501, torch.float16, 1), make([900], 513, 1501, torch.float16, 2)
    ya, yb = (torch.zeros((900, 513), device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    try:
        for _ in range(5):
            dev.set_stream(LEGACY)
            forward(wg, dev, *a, ya)
            dev.set_stream(s.cuda_stream)
            forward(wg, dev, *b, yb)
            dev.set_stream(None)
            forward(wg, dev, *a, ya)
    finally:
        torch.cuda.synchronize()
        dev.set_stream(LEGACY)
    for (x, w, off), y in ((a, ya), (b, yb)):
        want, mag = rows64(x, w, off)
        check(y, want, mag, 1501, "float32")


def test_threads_with_unaligned_operands(wg, dev):
    """Threads share a handle: each call's aligned copies stay with its own product."""
    import threading

    cases = [make([300 + i, 200], 257 + 2 * i, 1001 + 2 * i, torch.bfloat16, i) for i in range(4)]
    outs = [torch.zeros((500 + i, 257 + 2 * i), device="cuda") for i in range(4)]
    torch.cuda.synchronize()
    start, errors = threading.Barrier(4), []

    def work(i):
        try:
            start.wait()
            for _ in range(50):
                forward(wg, dev, *cases[i], outs[i])
        except Exception as e:  # noqa: BLE001 (reported below)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    torch.cuda.synchronize()
    dev.check()
    for (x, w, off), y in zip(cases, outs):
        want, mag = rows64(x, w, off)
        check(y, want, mag, x.shape[1], "float32")


# ---- values that must not spread ----------------------------------------------------------


def test_one_groups_infinities_stay_in_its_gradient(wg, dev):
    sizes = [70, 33, 1, 90]
    x, w, off = make(sizes, 264, 392)
    dy = torch.randn((194, 264), device="cuda").to(torch.bfloat16)
    x[70:103] = float("nan")
    dy[103] = float("inf")
    dw = torch.zeros((4, 264, 392), device="cuda")
    wg.gemmGroupedInner(dev, 4, 264, 392, 194, 1.0, dy, 264, x, 392, off, 0.0, dw, 392, 264 * 392)
    assert torch.isfinite(dw[[0, 3]]).all() and torch.isnan(dw[1]).all() and not torch.isfinite(dw[2]).any()


def test_beta_zero_does_not_read_c(wg, dev):
    x, w, off = make([70, 33], 136, 72)
    for dt in (torch.bfloat16, torch.float32):
        y = torch.full((103, 136), float("nan"), dtype=dt, device="cuda")
        forward(wg, dev, x, w, off, y)
        assert torch.isfinite(y).all()
    y = torch.full((103, 136), float("nan"), device="cuda")
    q, wq = wg.GpuMxMatrix.empty(dev, 103, 72), wg.GpuMxMatrix.empty(dev, 136, 72)
    wg.mxQuantize(dev, N, 103, 72, x, 72, q)
    wg.mxQuantize(dev, N, 136, 72, w, 72, wq)
    wg.mxGemm(dev, 103, 136, 72, 1.0, q, wq, 0.0, y, 136)
    assert torch.isfinite(y).all()
    q.destroy(), wq.destroy()


# ---- sizes past 32-bit offsets ----------------------------------------------------------------


def test_results_past_two_to_the_31_elements(wg, dev):
    m, n, k = 270000, 8192, 64
    x, w, off = make([m - 7, 7], n, k)
    y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    forward(wg, dev, x, w, off, y)
    for r in (slice(0, 40), slice(m - 300, m)):
        g = [0] * 40 if r.start == 0 else [0] * 293 + [1] * 7
        want = torch.stack([x[i].double() @ w[h].double().t() for i, h in zip(range(r.start, r.stop), g)])
        mag = torch.stack([x[i].double().abs() @ w[h].double().abs().t() for i, h in zip(range(r.start, r.stop), g)])
        check(y[r], want, mag, k, "bfloat16")


def test_as_many_rows_as_a_call_takes(wg, dev):
    m, n, k = (1 << 31) - 1025, 8, 8
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 70 GB of free device memory")
    x = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
    spots = [slice(0, 500), slice(1 << 30, (1 << 30) + 300), slice(m - 700, m)]
    for r in spots:
        x[r] = torch.randn((r.stop - r.start, k), device="cuda").to(torch.bfloat16)
    w = torch.randn((2, n, k), device="cuda").to(torch.bfloat16)
    forward(wg, dev, x, w, offsets_of([m - 5, 5]), y)
    dev.check()
    for r in spots:
        last = 5 if r.stop == m else 0
        want, mag = rows64(x[r], w, torch.tensor([0, r.stop - r.start - last, r.stop - r.start]))
        check(y[r], want, mag, k, "bfloat16")
    del x, y
    torch.cuda.empty_cache()


def test_weights_past_two_to_the_31_elements(wg, dev):
    groups, n, k = 40, 8192, 8192
    w = torch.zeros((groups, n, k), dtype=torch.bfloat16, device="cuda")
    w[0, :4], w[groups - 1] = torch.randn((4, k), device="cuda").bfloat16(), torch.randn((n, k), device="cuda").bfloat16()
    sizes = [2] + [0] * (groups - 2) + [3]
    x, off = torch.randn((5, k), device="cuda").bfloat16(), offsets_of(sizes)
    y = torch.zeros((5, n), device="cuda")
    forward(wg, dev, x, w, off, y)
    want, mag = rows64(x, w, off)
    check(y, want, mag, k, "float32")
    # the same in 4 bits, one matrix of the batch after the other
    wq, q = wg.GpuMxMatrix.empty(dev, n, k, batch=groups), wg.GpuMxMatrix.empty(dev, 5, k, groups=groups)
    wg.mxQuantize(dev, N, n, k, w, k, wq)
    wg.mxQuantize(dev, N, 5, k, x, k, q, offsets=off)
    wv = torch.empty((groups, n, k), dtype=torch.bfloat16, device="cuda")
    xv = torch.empty((5, k), dtype=torch.bfloat16, device="cuda")
    wg.mxDequantize(dev, wq, wv, k)
    wg.mxDequantize(dev, q, xv, k, offsets=off)
    wg.mxGemmGrouped(dev, groups, 5, n, k, 1.0, q, wq, off, 0.0, y, n)
    want, mag = rows64(xv, wv, off)
    check(y, want, mag, k, "float32")
    q.destroy(), wq.destroy()


def test_full_size(wg, dev):
    sizes = [1500, 0, 800, 1100, 37, 3000, 900, 855]
    n, k = 4096, 4096
    x, w, off = make(sizes, n, k)
    m = sum(sizes)
    y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    forward(wg, dev, x, w, off, y)
    want, mag = rows64(x, w, off)
    check(y, want, mag, k, "bfloat16")
    dw = torch.empty((8, n, k), device="cuda")
    dy = torch.randn((m, n), device="cuda").to(torch.bfloat16)
    wg.gemmGroupedInner(dev, 8, n, k, m, 1.0, dy, n, x, k, off, 0.0, dw, k, n * k)
    ends = off.tolist()
    for g in (0, 1, 4, 5):
        a, b = dy[ends[g]:ends[g + 1]].double(), x[ends[g]:ends[g + 1]].double()
        check(dw[g], a.t() @ b, a.abs().t() @ b.abs(), sizes[g], "float32")
        if sizes[g]:  # sums are drained: what truncation leaves is far below the bound
            e = (dw[g].double() - a.t() @ b).norm() / (a.t() @ b).norm()
            assert e < 1e-6


def test_full_size_in_4_bits(wg, dev):
    m, n, k = 4096, 8192, 4096
    x, w, off = make([m], n, k)
    xq, wq = wg.GpuMxMatrix.empty(dev, m, k), wg.GpuMxMatrix.empty(dev, n, k)
    wg.mxQuantize(dev, N, m, k, x, k, xq)
    wg.mxQuantize(dev, N, n, k, w, k, wq)
    y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    wg.mxGemm(dev, m, n, k, 1.0, xq, wq, 0.0, y, n)
    xv, wv = torch.empty((m, k), device="cuda"), torch.empty((n, k), device="cuda")
    wg.mxDequantize(dev, xq, xv, k)
    wg.mxDequantize(dev, wq, wv, k)
    want, mag = rows64(xv, wv[None], off)
    check(y, want, mag, k, "bfloat16")
    xq.destroy(), wq.destroy()


# ---- together ------------------------------------------------------------------------------------


def test_training_step_of_an_expert_layer(wg, dev):
    """Forward and both gradients of y = x W[g]^T, loss = sum(y * r): against the
    formulas in 64 bits, and against central differences of the 64-bit loss."""
    sizes, n, k = [120, 0, 77, 300, 1], 264, 392
    x, w, off = make(sizes, n, k)
    m = sum(sizes)
    r = torch.randn((m, n), device="cuda").to(torch.bfloat16)
    y = torch.empty((m, n), device="cuda")
    dx = torch.empty((m, k), device="cuda")
    dw = torch.zeros((5, n, k), device="cuda")
    forward(wg, dev, x, w, off, y)
    wg.gemmGrouped(dev, N, 5, m, k, n, 1.0, r, n, w, k, n * k, off, 0.0, dx, k)
    for part in range(2):  # gradient accumulation over two micro-batches, halves of each
        wg.gemmGroupedInner(dev, 5, n, k, m, 0.5, r, n, x, k, off, 1.0, dw, k, n * k)
    want, mag = rows64(x, w, off)
    check(y, want, mag, k, "float32")
    want, mag = rows64(r, w, off, trans=False)
    check(dx, want, mag, n, "float32")
    ends = off.tolist()
    for g in range(5):
        a, b = r[ends[g]:ends[g + 1]].double(), x[ends[g]:ends[g + 1]].double()
        check(dw[g], a.t() @ b, 2 * (a.abs().t() @ b.abs()), 2 * sizes[g] + 4, "float32")

    def loss(xx, ww):
        return sum((xx[ends[g]:ends[g + 1]] @ ww[g].t() * r[ends[g]:ends[g + 1]].double()).sum() for g in range(5))

    h = 2.0 ** -10
    vx, vw = torch.randn_like(x, dtype=torch.float64), torch.randn_like(w, dtype=torch.float64)
    x6, w6 = x.double(), w.double()
    dlx = (loss(x6 + h * vx, w6) - loss(x6 - h * vx, w6)) / (2 * h)
    dlw = (loss(x6, w6 + h * vw) - loss(x6, w6 - h * vw)) / (2 * h)
    # The loss is linear in each: the differences are exact up to 64-bit rounding; the
    # gradients' own error is that of fp32 sums.
    for got, d, v, terms in ((dx, dlx, vx, n), (dw, dlw, vw, max(sizes))):
        scale = (got.double() * v).abs().sum()
        assert ((got.double() * v).sum() - d).abs() <= terms * 2.0 ** -22 * scale


def test_serving_two_expert_layers_in_4_bits(wg, dev):
    """up = x Wu[g]^T, h = max(up, 0), down = h Wd[g]^T with all operands in MXFP4, for a
    prompt and then single tokens through the same weights."""
    groups, d, f = 4, 256, 520
    gen = torch.Generator(device="cuda").manual_seed(5)
    wu = torch.randn((groups, f, d), generator=gen, device="cuda").to(torch.bfloat16)
    wd = torch.randn((groups, d, f), generator=gen, device="cuda").to(torch.bfloat16)
    qu, qd = wg.GpuMxMatrix.empty(dev, f, d, batch=groups), wg.GpuMxMatrix.empty(dev, d, f, batch=groups)
    wg.mxQuantize(dev, N, f, d, wu, d, qu)
    wg.mxQuantize(dev, N, d, f, wd, f, qd)
    vu, vd = torch.empty_like(wu), torch.empty_like(wd)
    wg.mxDequantize(dev, qu, vu, d)
    wg.mxDequantize(dev, qd, vd, f)
    for sizes in ([130, 0, 41, 300], [0, 1, 0, 0], [1, 0, 2, 1]):
        m, off = sum(sizes), offsets_of(sizes)
        x = torch.randn((m, d), generator=gen, device="cuda").to(torch.bfloat16)
        up = torch.empty((m, f), dtype=torch.bfloat16, device="cuda")
        out = torch.empty((m, d), dtype=torch.bfloat16, device="cuda")
        qx, qh = wg.GpuMxMatrix.empty(dev, m, d, groups=groups), wg.GpuMxMatrix.empty(dev, m, f, groups=groups)
        wg.mxQuantize(dev, N, m, d, x, d, qx, offsets=off)
        wg.mxGemmGrouped(dev, groups, m, f, d, 1.0, qx, qu, off, 0.0, up, f)
        h = up.relu()
        wg.mxQuantize(dev, N, m, f, h, f, qh, offsets=off)
        wg.mxGemmGrouped(dev, groups, m, d, f, 1.0, qh, qd, off, 0.0, out, d)
        vx, vh = torch.empty_like(x), torch.empty_like(h)
        wg.mxDequantize(dev, qx, vx, d, offsets=off)
        wg.mxDequantize(dev, qh, vh, f, offsets=off)
        want, mag = rows64(vx, vu, off)
        check(up, want, mag, d, "bfloat16")
        want, mag = rows64(vh, vd, off)
        check(out, want, mag, f, "bfloat16")
        qx.destroy(), qh.destroy()
    dev.check()
    qu.destroy(), qd.destroy()


def test_gradients_of_a_linear_layer_in_4_bits(wg, dev):
    m, n, k = 300, 264, 520
    x, w, _ = make([m], n, k)
    dy = torch.randn((m, n), device="cuda").to(torch.bfloat16)
    mats = {}
    for name, t, src, r, c, ld in (("dy", N, dy, m, n, n), ("wt", T, w, k, n, k), ("dyt", T, dy, n, m, n), ("xt", T, x, k, m, k)):
        q = wg.GpuMxMatrix.empty(dev, r, c)
        wg.mxQuantize(dev, t, r, c, src, ld, q)
        v = torch.empty((r, c), dtype=torch.float32, device="cuda")
        wg.mxDequantize(dev, q, v, c)
        mats[name] = (q, v.double())
    dx, dw = torch.empty((m, k), dtype=torch.bfloat16, device="cuda"), torch.empty((n, k), device="cuda")
    wg.mxGemm(dev, m, k, n, 1.0, mats["dy"][0], mats["wt"][0], 0.0, dx, k)
    wg.mxGemm(dev, n, k, m, 1.0, mats["dyt"][0], mats["xt"][0], 0.0, dw, k)
    for got, a, b, terms, ct in ((dx, "dy", "wt", n, "bfloat16"), (dw, "dyt", "xt", m, "float32")):
        a, b = mats[a][1], mats[b][1]
        check(got, a @ b.t(), a.abs() @ b.abs().t(), terms, ct)
    # half a step of a 4-bit element is at most a sixth of it or an eighth of the block's scale limit
    assert ((mats["dy"][1] - dy.double()).norm() / dy.double().norm()) < 0.2
    for q, _ in mats.values():
        q.destroy()
