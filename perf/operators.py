"""The block-scaled operators as measured work: what a case is, its inputs, one pass, and what a pass cannot do without.

Block formats: a row is cut into blocks of 32 columns (the last one may be shorter) that share a power-of-two scale.

  4 bits   E = floor(log2 max|x|) - 2, element = x / 2^E rounded to nearest even on {0, .5, 1, 1.5, 2, 3, 4, 6},
           larger ones become 6; two to a byte (even column in the low half), 16 bytes a block
  8 bits   E = floor(log2 max|x|), element = round(64 x / 2^E) to nearest even in [-127, 127], value = element 2^(E-6)

and E (at least -127) is held as the byte E + 127.  Kinds of cases:

  quantize  x -> 4-bit blocks, and the values they stand for
  linear    y = f(x^ W^T + b), W in 4-bit blocks along its columns, f the identity or tanh, x^ = x or its 4-bit blocks; with
            "grad" also the gradients of x and b (the quantisation of x passes its gradient on unchanged)
  train     y = p(x) W + b, p the identity or tanh, and the gradients of x, W and b, for which the backward pass has x
            in 8-bit blocks only: gx = (g W^T) p'(x8), gW = p(x8)^T g, gb = sum g
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _kernels():
    package = os.path.abspath("flash-molecular-dynamics_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import flashmd_amd.kernels as kernels

    return kernels


# ---------------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one interaction layer's weights (128 x 128, the repository's model): the smallest call
        dict(name="quantize_layer", kind="quantize", dtype="fp32", m=128, k=128, data="weight"),
        # the radial basis of every edge of the 128-molecule benchmark batch: 50 columns, a short last block
        dict(name="quantize_basis", kind="quantize", dtype="fp32", m=1882048, k=50, data="basis"),
        # activations of a wide layer, 16 bits
        dict(name="quantize_wide", kind="quantize", dtype="bf16", m=8192, k=8192, data="normal"),
        # a single row through a wide layer: reading the weights is all there is
        dict(name="linear_one_row", kind="linear", dtype="bf16", m=1, k=4096, n=4096, tanh=False, bias=True, both=False,
             grad=False, data="normal"),
        # first filter layer over every edge of the benchmark batch, with the gradient that the forces need
        dict(name="linear_filter", kind="linear", dtype="fp32", m=1882048, k=50, n=128, tanh=True, bias=True, both=False,
             grad=True, data="basis"),
        # output network's first layer over the benchmark batch's beads, 16-bit activations, both operands in 4 bits
        dict(name="linear_output", kind="linear", dtype="fp16", m=34432, k=128, n=128, tanh=True, bias=True, both=True,
             grad=True, data="normal"),
        # odd sizes, weights only in 4 bits
        dict(name="linear_ragged", kind="linear", dtype="fp16", m=1111, k=1000, n=2001, tanh=False, bias=False, both=False,
             grad=True, data="normal"),
        # a large product of two 4-bit operands
        dict(name="linear_wide", kind="linear", dtype="bf16", m=8192, k=4096, n=8192, tanh=False, bias=True, both=True,
             grad=False, data="normal"),
        # one molecule of 269 beads: latency
        dict(name="train_molecule", kind="train", dtype="fp32", m=269, k=128, n=128, tanh=True, bias=True, data="normal"),
        # an interaction block's output layer over the benchmark batch
        dict(name="train_block", kind="train", dtype="fp32", m=34432, k=128, n=128, tanh=True, bias=True, data="normal"),
        # first filter layer over every edge of the benchmark batch
        dict(name="train_filter", kind="train", dtype="fp32", m=1882048, k=50, n=128, tanh=False, bias=True, data="basis"),
        # a wide layer in 16 bits
        dict(name="train_wide", kind="train", dtype="bf16", m=8192, k=4096, n=1024, tanh=True, bias=True, data="normal"),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 1e14


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("quantize", "linear", "train"))
        case = dict(kind=kind, dtype=rng.choice(tuple(DTYPES)))
        if rng.random() < 0.5:  # the layers of a model like this repository's, over few to very many rows
            case.update(m=_spread(rng, 1, 1900000), k=rng.randint(1, 160))
            n = rng.randint(1, 160)
        else:  # wide layers
            case.update(m=_spread(rng, 1, 8192), k=_spread(rng, 64, 8192))
            n = _spread(rng, 64, 8192)
        case["data"] = "basis" if case["k"] <= 64 and rng.random() < 0.5 else rng.choice(("normal", "weight"))
        if kind != "quantize":
            case.update(n=n, tanh=rng.random() < 0.5, bias=rng.random() < 0.7)
        if kind == "linear":
            case.update(both=rng.random() < 0.5, grad=rng.random() < 0.5)
        if _cost(case) <= limit:
            return case


def work(case):
    size = {"fp32": 4, "fp16": 2, "bf16": 2}[case["dtype"]]
    m, k = case["m"], case["k"]
    blocks = -(-k // BLOCK)
    if case["kind"] == "quantize":
        # x, the codes and scales, the values in 16 bits
        return {"bytes": m * k * size + m * blocks * 17 + m * k * 2, "flops": 4 * m * k}
    n = case["n"]
    bias = n * size if case["bias"] else 0
    if case["kind"] == "linear":
        weight = n * blocks * 17
        moved, flops = m * k * size + weight + bias + m * n * size, 2 * m * k * n
        if case["grad"]:  # g, gx and gb; the weights are there already
            moved += m * n * size + m * k * size + bias
            flops += 2 * m * k * n + (m * n if case["bias"] else 0)
        return {"bytes": moved, "flops": flops}
    # x, W, b, y; g, gx, gW, gb
    return {"bytes": 2 * m * k * size + 2 * m * n * size + 2 * k * n * size + 2 * bias, "flops": 6 * m * k * n + m * n}


# ---------------------------------------------------------------------------------------------------- inputs


def _values(data, m, k, gen):
    if data == "basis":  # Gaussians of a distance times the cosine cutoff, as the model's filter networks read them
        cutoff, spacing = 5.0, 5.0 / max(1, k - 1)
        distance = cutoff * torch.rand(m, 1, device="cuda", generator=gen) ** (1.0 / 3.0)
        centres = torch.arange(k, device="cuda", dtype=torch.float32) * spacing
        envelope = 0.5 * (torch.cos(distance * (math.pi / cutoff)) + 1.0)
        return torch.exp(-0.5 / spacing ** 2 * (distance - centres) ** 2) * envelope
    x = torch.randn(m, k, device="cuda", generator=gen)
    if data == "weight":  # Xavier's width
        return x * math.sqrt(1.0 / max(1, k))
    # features of unequal size, a few of them large
    return x * torch.exp(0.5 * torch.randn(1, k, device="cuda", generator=gen))


def _plain_quantize4(x):
    """(blocks of elements, exponents): x [m, k] in 32 bits -> [m, blocks, 32] on the grid, [m, blocks, 1] whole numbers."""
    m, k = x.shape
    blocks = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(m, -1, BLOCK)
    top = blocks.abs().amax(dim=2, keepdim=True)
    exponent = (torch.frexp(top)[1] - 3).clamp_min(-127)
    exponent = torch.where(top > 0, exponent, torch.full_like(exponent, -127))
    v = torch.ldexp(blocks, -exponent)
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return (torch.round(v / step) * step).clamp(-6, 6), exponent


def _plain_pack4(grid, exponent):
    """The bytes of 4-bit blocks: codes [m, 16 blocks], scales [m, blocks]."""
    size = grid.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    code = torch.where(size < 2, size / step, torch.where(size < 4, size / step + 2, size / step + 4)).to(torch.uint8)
    code = code | (torch.signbit(grid).to(torch.uint8) << 3)
    m = code.shape[0]
    return (code[..., 0::2] | (code[..., 1::2] << 4)).reshape(m, -1).contiguous(), (exponent[..., 0] + 127).to(torch.uint8)


def _plain_dequantize4(codes, scales, k, dtype=torch.float32):
    m = codes.shape[0]
    code = torch.stack((codes & 15, codes >> 4), dim=2).reshape(m, -1, BLOCK).long()
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device, dtype=dtype)
    return torch.ldexp(table[code], scales.int().unsqueeze(2) - 127).reshape(m, -1)[:, :k]


def _plain_blocks8(x):
    """x [m, k] in 32 bits -> the values of its 8-bit blocks."""
    m, k = x.shape
    blocks = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(m, -1, BLOCK)
    top = blocks.abs().amax(dim=2, keepdim=True)
    exponent = (torch.frexp(top)[1] - 1).clamp_min(-127)
    exponent = torch.where(top > 0, exponent, torch.full_like(exponent, -127))
    q = torch.round(torch.ldexp(blocks, -exponent) * 64).clamp(-127, 127)
    return torch.ldexp(q / 64, exponent).reshape(m, -1)[:, :k]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)
    dtype = DTYPES[case["dtype"]]
    m, k = case["m"], case["k"]
    state = dict(case, x=_values(case["data"], m, k, gen).to(dtype))
    if case["kind"] == "quantize":
        return state
    n = case["n"]
    weight = torch.randn(k, n, device="cuda", generator=gen) * math.sqrt(2.0 / (k + n))
    state["b"] = (0.1 * torch.randn(n, device="cuda", generator=gen)).to(dtype) if case["bias"] else None
    if case["kind"] == "linear":
        state["codes"], state["scales"] = _plain_pack4(*_plain_quantize4(weight.t().contiguous()))
    else:
        state["w"] = weight.to(dtype).requires_grad_()
    if case["kind"] == "train" or case["grad"]:
        state["g"] = (1e-3 * torch.randn(m, n, device="cuda", generator=gen)).to(dtype)
        state["x"].requires_grad_()
        if case["bias"]:
            state["b"].requires_grad_()
    return state


# ---------------------------------------------------------------------------------------------------- one pass


def _run_own(s):
    kernels = _kernels()
    if s["kind"] == "quantize":
        codes, scales = kernels.mxfp4_quantize(s["x"])
        return {"values": kernels.mxfp4_dequantize(codes, scales, s["k"], dtype=torch.bfloat16)}
    if s["kind"] == "linear":
        y = kernels.mxfp4_linear_autograd(s["x"], s["codes"], s["scales"], s["b"], activation="tanh" if s["tanh"] else None,
                                          quantize_input=s["both"])
        if not s["grad"]:
            return {"y": y}
        got = torch.autograd.grad(y, [t for t in (s["x"], s["b"]) if t is not None], s["g"])
        return {"y": y.detach(), "gx": got[0], "gb": got[1] if s["bias"] else None}
    layer = kernels.fused_tanh_linear_ckpt8_autograd if s["tanh"] else kernels.linear_ckpt8_autograd
    y = layer(s["x"], s["w"], s["b"])
    got = torch.autograd.grad(y, [t for t in (s["x"], s["w"], s["b"]) if t is not None], s["g"])
    return {"y": y.detach(), "gx": got[0], "gw": got[1], "gb": got[2] if s["bias"] else None}


def _run_plain(s):
    dtype, x = s["x"].dtype, s["x"].float()
    if s["kind"] == "quantize":
        grid, exponent = _plain_quantize4(x)
        codes, scales = _plain_pack4(grid, exponent)
        return {"values": _plain_dequantize4(codes, scales, s["k"]).bfloat16()}
    b = s["b"].float() if s["bias"] else None
    if s["kind"] == "linear":
        if s["both"]:
            grid, exponent = _plain_quantize4(x)
            x = torch.ldexp(grid, exponent).reshape(x.shape[0], -1)[:, :s["k"]]
        w = _plain_dequantize4(s["codes"], s["scales"], s["k"])
        y = x @ w.t()
        y = y + b if s["bias"] else y
        y = torch.tanh(y) if s["tanh"] else y
        if not s["grad"]:
            return {"y": y.to(dtype)}
        g = s["g"].float() * (1.0 - y * y) if s["tanh"] else s["g"].float()
        return {"y": y.to(dtype), "gx": (g @ w).to(dtype), "gb": g.sum(0).to(dtype) if s["bias"] else None}
    w, g, kept = s["w"].float(), s["g"].float(), _plain_blocks8(x)
    y = (torch.tanh(x) if s["tanh"] else x) @ w
    y = y + b if s["bias"] else y
    gx = g @ w.t()
    if s["tanh"]:
        kept = torch.tanh(kept)
        gx = gx * (1.0 - kept * kept)
    return {"y": y.to(dtype), "gx": gx.to(dtype), "gw": (kept.t() @ g).to(dtype), "gb": g.sum(0).to(dtype) if s["bias"] else None}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ---------------------------------------------------------------------------------------------------- in 64 bits


def _nearest(sizes, levels):
    """Each of `sizes` (none negative) to the nearest of the ascending `levels`, a tie to the one of even index."""
    found = torch.zeros_like(sizes)
    for i in range(1, len(levels)):
        middle = 0.5 * (levels[i - 1] + levels[i])
        found = torch.where((sizes > middle) | ((sizes == middle) & (i % 2 == 0)), levels[i], found)
    return found


def _exact_blocks(x, bits):
    """The values that the blocks of x [m, k], in 64 bits, stand for."""
    m, k = x.shape
    out = torch.empty_like(x)
    for a in range(0, k, BLOCK):
        part = x[:, a:a + BLOCK]
        top = part.abs().amax(1, keepdim=True)
        power = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
        power = torch.where(top >= torch.exp2(power + 1), power + 1, power)  # whatever log2 rounds to
        power = torch.where(top < torch.exp2(power), power - 1, power)
        scale = torch.exp2((power - (2 if bits == 4 else 0)).clamp_min(-127))
        scale = torch.where(top > 0, scale, 2.0 ** -127)
        if bits == 4:
            out[:, a:a + BLOCK] = torch.sign(part) * _nearest((part / scale).abs(), LEVELS) * scale
        else:
            out[:, a:a + BLOCK] = torch.round(part / scale * 64).clamp(-127, 127) / 64 * scale
    return out


def _exact_weight(codes, scales, k):
    code = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.int64, device=codes.device)
    code[:, 0::2], code[:, 1::2] = (codes % 16).long(), (codes // 16).long()
    size = torch.zeros(code.shape, dtype=torch.float64, device=codes.device)
    for i, level in enumerate(LEVELS):
        size[code % 8 == i] = level
    sign = torch.where(code >= 8, -1.0, 1.0).double()
    return (sign * size * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=1))[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        x = s["x"].double()
        if case["kind"] == "quantize":
            return {"values": _exact_blocks(x, 4)}
        b = s["b"].double() if case["bias"] else 0.0
        if case["kind"] == "linear":
            w = _exact_weight(s["codes"], s["scales"], case["k"])
            z = (_exact_blocks(x, 4) if case["both"] else x).matmul(w.t().contiguous()) + b
            y = torch.tanh(z) if case["tanh"] else z
            if not case["grad"]:
                return {"y": y}
            g = s["g"].double()
            if case["tanh"]:
                g = g / torch.cosh(z) ** 2
            return {"y": y, "gx": g.matmul(w), "gb": g.sum(0) if case["bias"] else None}
        w, g, kept = s["w"].double(), s["g"].double(), _exact_blocks(x, 8)
        y = (torch.tanh(x) if case["tanh"] else x).matmul(w) + b
        gx = g.matmul(w.t().contiguous())
        if case["tanh"]:
            gx = gx / torch.cosh(kept) ** 2
        gw = (torch.tanh(kept) if case["tanh"] else kept).t().contiguous().matmul(g)
        return {"y": y, "gx": gx, "gw": gw, "gb": g.sum(0) if case["bias"] else None}
