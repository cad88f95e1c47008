"""Block-scaled numbers and the layers on them in 64 bits, from their definition (test infrastructure only).

A row is cut into blocks of 32 columns with one exponent E; byte = E + 127, 255 for a block that holds an Inf or a NaN.
  4 bits: E = max(floor(log2 amax) - 2, -127), x / 2^E to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (a tie to the even code)
  8 bits: E = max(floor(log2 amax), -127), code = nearest even of 64 x / 2^E within +-127, value = code 2^(E-6)
"""
from __future__ import annotations

import math

import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _blocks(x: torch.Tensor):
    """(blocks [m, nb, 32] in 64 bits, E [m, nb], bad [m, nb])"""
    m, k = x.shape
    nb = -(-k // 32)
    b = torch.zeros(m, nb * 32, dtype=torch.float64)
    b[:, :k] = x.double()
    b = b.view(m, nb, 32)
    bad = ~torch.isfinite(b).all(dim=2)
    top = torch.where(bad, torch.zeros(()).double(), b.abs().amax(dim=2)) if m else torch.zeros(m, nb, dtype=torch.float64)
    e = torch.tensor([[math.frexp(v)[1] - 1 if v > 0 else -10000 for v in row] for row in top.tolist()], dtype=torch.int64)
    return torch.where(bad.unsqueeze(2), torch.zeros(()).double(), b), e.view(m, nb), bad


def _scaled(b, e):
    """b / 2^e without an overflowing power"""
    half = torch.div(e, 2, rounding_mode="floor")
    return b * torch.exp2(-half.double()).unsqueeze(2) * torch.exp2(-(e - half).double()).unsqueeze(2)


def _values(q, e, bad, k):
    v = q * torch.exp2(e.double()).unsqueeze(2)
    v[bad] = float("nan")
    return v.reshape(v.shape[0], -1)[:, :k]


def mxfp4(x: torch.Tensor):
    """(codes uint8 [m, 16 nb], scales uint8 [m, nb], values [m, k] in 64 bits)"""
    b, e, bad = _blocks(x)
    e = (e - 2).clamp_min(-127)
    v = _scaled(b, e)
    code = torch.zeros(v.shape, dtype=torch.int64)
    for i in range(1, 8):
        mid = 0.5 * (LEVELS[i - 1] + LEVELS[i])
        code[(v.abs() > mid) | ((v.abs() == mid) & torch.tensor(i % 2 == 0))] = i
    code[torch.signbit(b)] += 8
    code[bad] = 0
    q = torch.tensor(LEVELS, dtype=torch.float64)[code % 8] * torch.where(code >= 8, -1.0, 1.0).double()
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    flat = code.reshape(code.shape[0], -1)
    return (flat[:, 0::2] + 16 * flat[:, 1::2]).to(torch.uint8), scales, _values(q, e, bad, x.shape[1])


def mxint8(x: torch.Tensor):
    """(codes int8 [m, 32 nb], scales uint8 [m, nb], values [m, k] in 64 bits)"""
    b, e, bad = _blocks(x)
    e = e.clamp_min(-127)
    q = torch.round(_scaled(b, e) * 64).clamp(-127, 127)
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return q.reshape(q.shape[0], -1).to(torch.int8), scales, _values(q / 64, e, bad, x.shape[1])


def linear(x, w, bias=None, tanh=False, both=False, g=None):
    """y = f(x^ w^T + b), w [n, k] values in 64 bits; with g also (gx, gb)"""
    x = mxfp4(x)[2] if both else x.double()
    z = x @ w.t().contiguous() + (0.0 if bias is None else bias.double())
    y = torch.tanh(z) if tanh else z
    if g is None:
        return y
    gz = g.double() / torch.cosh(z) ** 2 if tanh else g.double()
    return y, gz @ w, gz.sum(0)


def linear_ckpt8(x, w, bias=None, tanh=False, g=None):
    """y = p(x) w + b, w [k, n]; with g also (gx, gw, gb) from x's 8-bit blocks"""
    w, kept = w.double(), mxint8(x)[2]
    p = torch.tanh if tanh else (lambda t: t)
    y = p(x.double()) @ w + (0.0 if bias is None else bias.double())
    if g is None:
        return y
    g = g.double()
    gx = g @ w.t().contiguous()
    if tanh:
        gx = gx / torch.cosh(kept) ** 2
    return y, gx, p(kept).t().contiguous() @ g, g.sum(0)
