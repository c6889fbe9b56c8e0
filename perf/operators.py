"""Cases of the expert-grouped and microscaled (MXFP4) products, for timing and comparison.

``run`` computes a case either in its plain form (elementary torch operations in
32 bits) or, where ``own`` is true, through wgblas_b200's public calls
(``gemmGrouped``, ``gemmGroupedInner``, ``mxQuantize``, ``mxDequantize``,
``mxGemm``, ``mxGemmGrouped``). ``exact`` gives the same outputs from the
operators' definitions in 64 bits.

The operators, with rows of X sorted by expert and row range offsets[g] ..
offsets[g + 1] belonging to expert g:

* grouped:       Y[r] = W[g] X[r]                       (W[g]: n x k)
* grouped_grad:  dX[r] = W[g]^T dY[r],  dW[g] = sum over r of dY[r] X[r]^T
* quantize:      X -> blocks of 32 along a row, a power-of-two scale for each
                 (2^(floor(log2 max|x|) - 2)), elements rounded to
                 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives, ties to even, above 6 to 6;
                 returned as the values they stand for
* mx:            Y = quantize(X) Wq^T, with the weights Wq held in MXFP4
* mx_grad:       dX = quantize(dY) quantize(W^T)^T, dW = quantize(dY^T) quantize(X^T)^T
* mx_grouped:    Y[r] = Wq[g] quantize(X)[r]
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One token in the air, routed to four of eight small experts: launch latency.
        {"name": "grouped one token", "op": "grouped", "m": 4, "n": 512, "k": 1024, "groups": 8, "type": "bf16"},
        # A decoding batch: every expert's weights are read for a few tokens each.
        {"name": "grouped decode", "op": "grouped", "m": 256, "n": 2048, "k": 2048, "groups": 64, "type": "bf16"},
        # A long prompt through wide experts: bound by the tensor cores.
        {"name": "grouped prompt", "op": "grouped", "m": 16384, "n": 4096, "k": 4096, "groups": 16, "type": "bf16"},
        # Sizes that no vector load divides, and rows behind the last expert's.
        {"name": "grouped odd", "op": "grouped", "m": 1000, "n": 1023, "k": 777, "groups": 7, "type": "fp16",
         "unused": 5},
        # The backward pass of an expert layer in training, weight gradients in 32 bits.
        {"name": "grouped gradients", "op": "grouped_grad", "m": 8192, "n": 2048, "k": 4096, "groups": 8,
         "type": "bf16"},
        # The same with ragged, unaligned sizes and half precision.
        {"name": "grouped gradients odd", "op": "grouped_grad", "m": 1111, "n": 514, "k": 1002, "groups": 19,
         "type": "fp16"},
        # A whole activation or weight matrix through the format: bound by memory.
        {"name": "quantize matrix", "op": "quantize", "m": 8192, "k": 8192, "type": "bf16"},
        # One ragged handful of rows in 32 bits.
        {"name": "quantize rows", "op": "quantize", "m": 33, "k": 1023, "type": "fp32"},
        # A linear layer's forward over a prompt, weights kept in 4 bits.
        {"name": "mx prompt", "op": "mx", "m": 8192, "n": 8192, "k": 4096, "type": "bf16"},
        # The same layer for a few tokens: the weights' bytes and two launches.
        {"name": "mx decode", "op": "mx", "m": 16, "n": 8192, "k": 4096, "type": "bf16"},
        # Both gradients of a linear layer in 4-bit arithmetic.
        {"name": "mx gradients", "op": "mx_grad", "m": 4096, "n": 4096, "k": 2048, "type": "bf16"},
        # Experts with weights in 4 bits over a serving batch.
        {"name": "mx experts", "op": "mx_grouped", "m": 1500, "n": 2048, "k": 4096, "groups": 32, "type": "bf16"},
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of the range; one in three a multiple of 64, one in three even."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    step = rng.choice((1, 2, 64))
    return max(low, v // step * step)


def draw(rng):
    op = rng.choice(("grouped", "grouped", "grouped_grad", "quantize", "mx", "mx_grad", "mx_grouped"))
    case = {"op": op, "m": _size(rng, 1, 16384), "k": _size(rng, 32, 4096)}
    if op == "quantize":
        return dict(case, type=rng.choice(("bf16", "fp32")))
    case["n"] = _size(rng, 32, 4096)
    if op.startswith("grouped") or op == "mx_grouped":
        # The experts' weights stay within half a gigaelement.
        case["groups"] = _size(rng, 1, max(1, min(128, (1 << 29) // (case["n"] * case["k"]))))
        case["unused"] = rng.choice((0, 0, min(3, case["m"] - 1)))
    if op.endswith("grad"):
        case["m"] = min(case["m"], 8192)
    case["type"] = rng.choice(("bf16", "bf16", "fp16")) if op.startswith("grouped") else "bf16"
    return case


# ---- inputs --------------------------------------------------------------------


def _sizes(case, gen):
    """Row counts of the experts: popular and unpopular ones, at times one with no rows."""
    g, rows = case["groups"], case["m"] - case.get("unused", 0)
    weight = torch.softmax(0.5 * torch.randn(g, generator=gen), 0)
    if rows == 0:
        return torch.zeros(g, dtype=torch.int64)
    taken = torch.multinomial(weight, rows, replacement=True, generator=gen)
    return torch.bincount(taken, minlength=g)


def _normal(shape, gen, dtype, scale=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    step = max(1, (1 << 28) // max(1, math.prod(shape[1:])))
    for i in range(0, shape[0], step):  # in pieces, so that no 32-bit copy of a whole stack is made
        out[i:i + step] = torch.randn(out[i:i + step].shape, generator=gen, device="cuda").mul_(scale)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dtype, m, k = _TYPES[case["type"]], case["m"], case["k"]
    s = {"case": case}
    # Activations: a few channels are far larger than the rest, as trained models have them.
    channel = torch.exp(0.7 * torch.randn(k, generator=gen, device="cuda"))
    s["X"] = (torch.randn((m, k), generator=gen, device="cuda") * channel).to(dtype)
    if case["op"] == "quantize":
        s["out"] = torch.empty_like(s["X"])
        s["work"] = _mx_room(m, k)
        return s
    n = case["n"]
    if "groups" in case:
        sizes = _sizes(case, host)
        s["most"] = max(1, int(sizes.max()))
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).to(torch.int32).cuda()
    if case["op"] == "grouped":
        s["W"] = _normal((case["groups"], n, k), gen, dtype, k ** -0.5)
        s["Y"] = torch.zeros((m, n), dtype=dtype, device="cuda")
    elif case["op"] == "grouped_grad":
        s["W"] = _normal((case["groups"], n, k), gen, dtype, k ** -0.5)
        s["dY"] = _normal((m, n), gen, dtype)
        s["dX"] = torch.zeros((m, k), dtype=dtype, device="cuda")
        s["dW"] = torch.zeros((case["groups"], n, k), dtype=torch.float32, device="cuda")
    elif case["op"] == "mx_grad":
        s["W"] = _normal((n, k), gen, dtype, k ** -0.5)
        s["dY"] = _normal((m, n), gen, dtype)
        s["dX"] = torch.empty((m, k), dtype=dtype, device="cuda")
        s["dW"] = torch.empty((n, k), dtype=torch.float32, device="cuda")
        # Room for the four quantised operands, kept by the training loop.
        s["work"] = [_mx_room(m, n), _mx_room(k, n), _mx_room(n, m), _mx_room(k, m)]
    else:
        stack = (case.get("groups", 1), n, k)
        s["Wq"] = _mx_pack(_normal(stack, gen, dtype, k ** -0.5))
        s["Y"] = torch.zeros((m, n), dtype=dtype, device="cuda")
        s["work"] = _mx_room(m, k, case.get("groups", 0))
    return s


def _mx_room(rows, cols, groups=0):
    """Memory for a quantised rows x cols matrix: 16 bytes of codes for each block of
    32, and the scales in tiles of 128 rows x 4 blocks (each expert begins a tile)."""
    codes = torch.zeros((rows, -(-cols // 32) * 16), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((-(-rows // 128) + groups) * -(-cols // 128) * 512, dtype=torch.uint8, device="cuda")
    return codes, scales


def _mx_pack(w):
    """A stack of weights as they are stored: two codes a byte (the even element in the
    low half), and 8-bit scale exponents in tiles of 128 rows x 4 blocks, where row r's
    four bytes stand at 16 * (r % 32) + 4 * (r // 32)."""
    batch, rows, cols = w.shape
    codes = torch.empty((batch, rows, -(-cols // 32) * 16), dtype=torch.uint8, device="cuda")
    tall, wide = -(-rows // 128), -(-cols // 128)
    scales = torch.zeros((batch, tall * 128, wide * 4), dtype=torch.uint8, device="cuda")
    lut = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], dtype=torch.uint8, device="cuda")
    for i in range(batch):
        q, e = _mx_round(w[i].float())
        c = lut[(q.abs() * 2).long()] + 8 * torch.signbit(q).to(torch.uint8)
        c = c.reshape(rows, -1, 2)
        codes[i] = c[..., 0] + 16 * c[..., 1]
        scales[i, :rows, : e.shape[1]] = (e[..., 0] + 127).to(torch.uint8)
    tiles = scales.reshape(batch, tall, 4, 32, wide, 4).permute(0, 1, 4, 3, 2, 5)
    return codes, tiles.contiguous().reshape(-1)


# ---- the plain form -----------------------------------------------------------------


def _two(e):
    """2^e in 32 bits, from its bit pattern (-127 is the one subnormal)."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _mx_round(x):
    """(elements, exponents) of x in blocks of 32 along its last axis, padded with zeros."""
    pad = -x.shape[-1] % 32
    if pad:
        x = torch.cat([x, x.new_zeros(*x.shape[:-1], pad)], -1)
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(-127, 127)
    a = b.abs() * _two(-e)
    q = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2))
    return torch.copysign(q.clamp(max=6), b), e


def _mx_values(x):
    q, e = _mx_round(x)
    return (q * _two(e)).reshape(*x.shape[:-1], -1)[..., : x.shape[-1]]


def _mx_unpack(packed, rows, cols):
    """The values that stored weights stand for."""
    codes, scales = packed
    batch, tall, wide = codes.shape[0], -(-rows // 128), -(-cols // 128)
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    q = lut[torch.stack([codes & 15, codes >> 4], -1).int()].reshape(batch, rows, -1, 32)
    e = scales.reshape(batch, tall, wide, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(batch, tall * 128, wide * 4)
    e = e[:, :rows, : q.shape[2], None].int() - 127
    return (q * _two(e)).reshape(batch, rows, -1)[..., :cols]


def _stacked(s, x):
    """x's rows by expert in 32 bits, each padded with zeros to the largest: groups x most x width."""
    at = s["offsets"][:-1, None].long() + torch.arange(s["most"], device="cuda")
    inside = at < s["offsets"][1:, None]
    return torch.where(inside[..., None], x[at.clamp(max=x.shape[0] - 1)].float(), 0.0)


def _unstacked(s, y, like):
    """The rows of `y` (groups x most x width) back in their places; the other rows as in `like`."""
    row = torch.arange(like.shape[0], device="cuda")
    g = torch.searchsorted(s["offsets"][1:].long(), row, right=True).clamp(max=y.shape[0] - 1)
    pos = (row - s["offsets"].long()[g]).clamp(max=y.shape[1] - 1)
    return torch.where((row < s["offsets"][-1])[:, None], y[g, pos].to(like.dtype), like)


def _plain(s):
    op, case = s["case"]["op"], s["case"]
    if op == "grouped":
        y = torch.bmm(_stacked(s, s["X"]), s["W"].float().transpose(1, 2))
        return _unstacked(s, y, torch.zeros_like(s["Y"]))
    if op == "grouped_grad":
        dy = _stacked(s, s["dY"])
        dw = torch.bmm(dy.transpose(1, 2), _stacked(s, s["X"]))
        dx = _unstacked(s, torch.bmm(dy, s["W"].float()), torch.zeros_like(s["dX"]))
        return {"dX": dx, "dW": dw}
    if op == "quantize":
        return _mx_values(s["X"].float()).to(s["X"].dtype)
    if op == "mx":
        w = _mx_unpack(s["Wq"], case["n"], case["k"])[0]
        return (_mx_values(s["X"].float()) @ w.t()).to(s["X"].dtype)
    if op == "mx_grad":
        x, w, dy = s["X"].float(), s["W"].float(), s["dY"].float()
        dx = _mx_values(dy) @ _mx_values(w.t()).t()
        dw = _mx_values(dy.t()) @ _mx_values(x.t()).t()
        return {"dX": dx.to(s["X"].dtype), "dW": dw}
    w = _mx_unpack(s["Wq"], case["n"], case["k"])
    y = torch.bmm(_stacked(s, _mx_values(s["X"].float())), w.transpose(1, 2))
    return _unstacked(s, y, torch.zeros_like(s["Y"]))


# ---- the framework's calls -------------------------------------------------------------

_device = None


def _gpu(wg):
    """The program's device handle, its work ordered on torch's default stream (the legacy stream, handle 1)."""
    global _device
    if _device is None:
        _device = wg.init()
        _device.set_stream(1)
    return _device


def _own(s):
    import wgblas_b200 as wg

    dev, case, op = _gpu(wg), s["case"], s["case"]["op"]
    m, k, n, groups = case["m"], case["k"], case.get("n", 0), case.get("groups", 0)
    if op == "grouped":
        wg.gemmGrouped(dev, "transpose", groups, m, n, k, 1.0, s["X"], k, s["W"], k, n * k, s["offsets"], 0.0,
                       s["Y"], n)
        return s["Y"]
    if op == "grouped_grad":
        wg.gemmGrouped(dev, "no-transpose", groups, m, k, n, 1.0, s["dY"], n, s["W"], k, n * k, s["offsets"], 0.0,
                       s["dX"], k)
        wg.gemmGroupedInner(dev, groups, n, k, m, 1.0, s["dY"], n, s["X"], k, s["offsets"], 0.0, s["dW"], k, n * k)
        return {"dX": s["dX"], "dW": s["dW"]}
    if op == "quantize":
        q = wg.GpuMxMatrix.wrap(dev, *s["work"], m, k)
        wg.mxQuantize(dev, "no-transpose", m, k, s["X"], k, q)
        wg.mxDequantize(dev, q, s["out"], k)
        return s["out"]
    if op == "mx":
        q = wg.GpuMxMatrix.wrap(dev, *s["work"], m, k)
        w = wg.GpuMxMatrix.wrap(dev, *s["Wq"], n, k)
        wg.mxQuantize(dev, "no-transpose", m, k, s["X"], k, q)
        wg.mxGemm(dev, m, n, k, 1.0, q, w, 0.0, s["Y"], n)
        return s["Y"]
    if op == "mx_grad":
        dy, wt, dyt, xt = (wg.GpuMxMatrix.wrap(dev, *room, *shape)
                           for room, shape in zip(s["work"], ((m, n), (k, n), (n, m), (k, m))))
        wg.mxQuantize(dev, "no-transpose", m, n, s["dY"], n, dy)
        wg.mxQuantize(dev, "transpose", k, n, s["W"], k, wt)
        wg.mxQuantize(dev, "transpose", n, m, s["dY"], n, dyt)
        wg.mxQuantize(dev, "transpose", k, m, s["X"], k, xt)
        wg.mxGemm(dev, m, k, n, 1.0, dy, wt, 0.0, s["dX"], k)
        wg.mxGemm(dev, n, k, m, 1.0, dyt, xt, 0.0, s["dW"], k)
        return {"dX": s["dX"], "dW": s["dW"]}
    q = wg.GpuMxMatrix.wrap(dev, *s["work"], m, k, groups=groups)
    w = wg.GpuMxMatrix.wrap(dev, *s["Wq"], n, k, batch=groups)
    wg.mxQuantize(dev, "no-transpose", m, k, s["X"], k, q, offsets=s["offsets"])
    wg.mxGemmGrouped(dev, groups, m, n, k, 1.0, q, w, s["offsets"], 0.0, s["Y"], n)
    return s["Y"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a case costs ---------------------------------------------------------------------


def _touched(case):
    """Experts that are expected to have rows."""
    g, rows = case["groups"], case["m"] - case.get("unused", 0)
    return g * (1 - (1 - 1 / g) ** rows)


def work(case):
    m, k, e, op = case["m"], case["k"], _BYTES[case["type"]], case["op"]
    mx = 0.5 + 1 / 32  # bytes of an element in 4 bits with its share of a scale
    if op == "quantize":  # into the format and out of it again
        return {"bytes": 2.0 * m * k * (e + mx), "flops": 4.0 * m * k}
    n = case["n"]
    if op == "grouped":
        return {"bytes": float(e * (m * k + m * n + _touched(case) * n * k)), "flops": 2.0 * m * n * k}
    if op == "grouped_grad":
        return {"bytes": float(e * (2 * m * k + m * n + _touched(case) * n * k) + 4 * case["groups"] * n * k),
                "flops": 4.0 * m * n * k}
    if op == "mx_grad":
        return {"bytes": float(e * (2 * m * k + m * n + n * k) + 4 * n * k), "flops": 4.0 * m * n * k}
    w = (_touched(case) if op == "mx_grouped" else 1) * n * k * mx
    return {"bytes": float(e * (m * k + m * n) + w), "flops": 2.0 * m * n * k}


# ---- the definition in 64 bits ---------------------------------------------------------------


def _exact_mx(x):
    """The values of x in MXFP4, by distance to the eight magnitudes (ties to the even code)."""
    x = x.double()
    cols = x.shape[1]
    out = torch.zeros((x.shape[0], -(-cols // 32) * 32), dtype=torch.float64, device="cuda")
    out[:, :cols] = x
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    middle = (grid[1:] + grid[:-1]) / 2
    table = torch.tensor([2.0 ** e for e in range(-127, 128)], dtype=torch.float64, device="cuda")
    step = max(1, (1 << 24) // out.shape[1])
    for i in range(0, out.shape[0], step):
        b = out[i:i + step].unflatten(1, (-1, 32))
        top = b.abs().max(dim=2, keepdim=True).values
        # the largest table entry 2^e with 4 * 2^e <= max|x|, the smallest where there is none
        scale = table[(torch.searchsorted(4 * table, top, right=True) - 1).clamp(min=0)]
        a = b.abs() / scale
        up, down = torch.searchsorted(middle, a, right=True), torch.searchsorted(middle, a, right=False)
        code = torch.where(up == down, up, torch.where(up % 2 == 0, up, down))
        out[i:i + step] = (torch.sign(b) * grid[code] * scale).flatten(1)
    return out[:, :cols]


def _exact_stored(packed, g, rows, cols):
    """Expert g's stored weights, gathered element by element from their codes and scale tiles."""
    codes, scales = packed
    r = torch.arange(rows, device="cuda")[:, None]
    c = torch.arange(cols, device="cuda")[None, :]
    nibble = (codes[g][r, c // 2].int() >> (4 * (c % 2))) & 15
    mag, sign = nibble & 7, nibble >> 3
    # 1 exponent bit pattern: 0 and 1 are 0 and 0.5, the others (1 + m / 2) * 2^(e - 1)
    power = torch.tensor([2.0 ** e for e in range(-127, 129)], dtype=torch.float64, device="cuda")
    value = torch.where(mag < 2, mag * 0.5, (1 + 0.5 * (mag % 2)) * power[mag // 2 + 126])
    tile = (g * -(-rows // 128) + r // 128) * -(-cols // 128) + c // 128
    byte = tile * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c // 32 % 4
    return value.double() * (1 - 2 * sign) * power[scales[byte].int()]


def exact(case, seed):
    s = prepare(case, seed)
    op, k = case["op"], case["k"]
    if op == "quantize":
        return _exact_mx(s["X"])
    if op == "mx":
        return _exact_mx(s["X"]) @ _exact_stored(s["Wq"], 0, case["n"], k).t()
    if op == "mx_grad":
        dx = _exact_mx(s["dY"]) @ _exact_mx(s["W"].t()).t()
        return {"dX": dx, "dW": _exact_mx(s["dY"].t()) @ _exact_mx(s["X"].t()).t()}
    ends = s["offsets"].tolist()
    if op == "grouped_grad":
        dx = torch.zeros(s["dX"].shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros(s["dW"].shape, dtype=torch.float64, device="cuda")
        for g in range(case["groups"]):
            rows = slice(ends[g], ends[g + 1])
            dx[rows] = s["dY"][rows].double() @ s["W"][g].double()
            dw[g] = s["dY"][rows].double().t() @ s["X"][rows].double()
        return {"dX": dx, "dW": dw}
    x = s["X"].double() if op == "grouped" else _exact_mx(s["X"])
    y = torch.zeros(s["Y"].shape, dtype=torch.float64, device="cuda")
    for g in range(case["groups"]):
        rows = slice(ends[g], ends[g + 1])
        if ends[g] < ends[g + 1]:
            w = s["W"][g].double() if op == "grouped" else _exact_stored(s["Wq"], g, case["n"], k)
            y[rows] = x[rows] @ w.t()
    return y
