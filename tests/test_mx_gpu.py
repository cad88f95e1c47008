"""Block-scaled layers on the GPU against the 64-bit oracle (oracle/mx_oracle.py).

Codes and scales are compared bit for bit: scaling by a power of two is exact, so they are functions of the input's bits.

Tolerances (relative 2-norm), u = half a step of the type (``torch.finfo(t).eps / 2``):
  32 bits: operands are exact sums of bf16 planes and at most 6 plane products a term are summed in fp32, so what is left is
    the sums' rounding.  An addition is off by at most u of the partial sum; n of them in random directions by u sqrt(n), and
    a tanh or its derivative adds a few u: 2^-24 (8 + 2 sqrt(6 terms)), twice the random walk.
  16 bits: the output's rounding (u), and one for each operand that is computed before the product (u each): at most 3 u.
"""
import pytest
import torch

from oracle import mx_oracle as mo

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def K():
    import flashmd_amd.kernels as kernels

    assert torch.cuda.is_available(), "these tests need the MI355X"
    return kernels


def tolerance(dtype, terms):
    wide = 2.0 ** -24 * (8 + 2 * (6 * max(1, terms)) ** 0.5)
    return wide if dtype == torch.float32 else wide + 3 * torch.finfo(dtype).eps / 2


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape
    return float((a - b).norm() / b.norm().clamp_min(1e-30)) if a.numel() else 0.0


def near(a, b, terms, what=""):
    r, tol = rel(a, b), tolerance(a.dtype, terms)
    assert r <= tol, f"{what}: {r:.3g} > {tol:.3g}"


def rand(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def uneven(m, k, dtype, seed=0):
    """rows and columns of very different size, zeros among them"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(2.0 * torch.randn(m, 1, generator=g)) * torch.exp(torch.randn(1, k, generator=g))
    x[torch.rand(m, k, generator=g) < 0.1] = 0.0
    return x.to(dtype)


# ---------------------------------------------------------------------------------------- the formats
SHAPES = [(1, 1), (3, 31), (5, 32), (7, 33), (9, 50), (64, 128), (129, 200), (2, 1000), (300, 7)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_bit_exact(K, shape, dtype):
    x = uneven(*shape, dtype, seed=shape[1])
    for quantize, dequantize, oracle in ((K.mxfp4_quantize, K.mxfp4_dequantize, mo.mxfp4), (K.mxint8_quantize, K.mxint8_dequantize, mo.mxint8)):
        codes, scales, values = oracle(x)
        c, s = quantize(x.to(DEV))
        assert c.dtype == codes.dtype and torch.equal(c.cpu(), codes) and torch.equal(s.cpu(), scales)
        for out in (torch.float32, torch.bfloat16):
            assert torch.equal(dequantize(c, s, shape[1], dtype=out).cpu().double(), values)
        assert torch.equal(dequantize(c, s, shape[1], dtype=torch.float16).cpu(), values.half())


def test_quantize_special_rows(K):
    inf, nan = float("inf"), float("nan")
    grid = torch.arange(0, 8.01, 0.125)                      # ties and saturation of both signs, amax in [4, 8)
    rows = [torch.cat((grid[:31], torch.tensor([7.99]))), -torch.cat((grid[32:63], torch.tensor([4.0]))),
            torch.zeros(32), -torch.zeros(32), torch.full((32,), 3.4e38), torch.full((32,), 1e-45), torch.linspace(-1.2e-38, 1e-38, 32),
            torch.linspace(-3e-38, 2e-38, 32), torch.tensor([0.0, inf] + [1.0] * 30), torch.tensor([nan] * 32),
            torch.tensor([-inf] + [0.0] * 31), torch.tensor([1.0] * 31 + [nan]), torch.tensor([2.0 ** -126] + [2.0 ** -130] * 31),
            torch.tensor([127.0 / 64, 127.5 / 64, -127.5 / 64, 0.5 / 64, 1.5 / 64, 2.5 / 64, -0.5 / 64] + [1.0] * 25)]
    x = torch.stack(rows)
    for quantize, dequantize, oracle in ((K.mxfp4_quantize, K.mxfp4_dequantize, mo.mxfp4), (K.mxint8_quantize, K.mxint8_dequantize, mo.mxint8)):
        codes, scales, values = oracle(x)
        c, s = quantize(x.to(DEV))
        assert torch.equal(c.cpu(), codes) and torch.equal(s.cpu(), scales)
        assert torch.equal(torch.nan_to_num(dequantize(c, s, 32).cpu().double(), nan=-1.25), torch.nan_to_num(values, nan=-1.25))


def test_quantize_empty_and_views(K):
    c, s = K.mxfp4_quantize(torch.empty(0, 40, device=DEV))
    assert c.shape == (0, 32) and s.shape == (0, 2) and K.mxfp4_dequantize(c, s, 40).shape == (0, 40)
    flat = rand(7 * 40 + 1, seed=4).to(DEV)
    x = flat[1:].view(7, 40)                                 # not on a 16-byte boundary
    assert torch.equal(K.mxfp4_quantize(x)[0].cpu(), mo.mxfp4(x.cpu())[0])
    assert torch.equal(K.mxint8_quantize(x)[0].cpu(), mo.mxint8(x.cpu())[0])


# ---------------------------------------------------------------------------------------- 4-bit layers
LAYERS = [(1, 1, 1), (1, 50, 128), (2, 33, 7), (3, 128, 64), (17, 64, 1), (32, 300, 130), (33, 31, 128), (64, 128, 128), (100, 129, 33),
          (269, 50, 128), (269, 128, 64), (300, 256, 257), (1000, 128, 128), (65, 1000, 300)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("m,k,n", LAYERS)
def test_mxfp4_linear(K, m, k, n, both, dtype):
    x = uneven(m, k, dtype, seed=m + k)
    codes, scales, w = mo.mxfp4(rand(n, k, seed=n, scale=(2.0 / (k + n)) ** 0.5))
    bias, g = rand(n, seed=2, dtype=dtype), rand(m, n, seed=3, scale=1e-2, dtype=dtype)
    c, s, b = codes.to(DEV), scales.to(DEV), bias.to(DEV)
    for activation, with_bias in ((None, False), (None, True), ("tanh", True)):
        use = bias if with_bias else None
        y_ref, gx_ref, gb_ref = mo.linear(x, w, use, activation == "tanh", both, g)
        xg = x.to(DEV).requires_grad_()
        bg = b.clone().requires_grad_() if with_bias else None
        y = K.mxfp4_linear_autograd(xg, c, s, bg, activation, quantize_input=both)
        assert y.dtype == dtype
        near(y, y_ref, k, "y")
        assert torch.equal(y, K.mxfp4_linear(xg.detach(), c, s, None if bg is None else bg.detach(), activation, quantize_input=both))
        got = torch.autograd.grad(y, [xg] + ([bg] if with_bias else []), g.to(DEV))
        assert got[0].dtype == dtype
        near(got[0], gx_ref, n, "gx")
        if with_bias:
            near(got[1], gb_ref, m, "gb")


@pytest.mark.parametrize("both", [False, True])
def test_mxfp4_linear_weight_codes_behind_the_last_column_do_not_matter(K, both):
    """k = 40: the second block's codes behind column 8 hold anything, the result is that of zeros."""
    m, k, n = 37, 40, 50
    x = rand(m, k, seed=1)
    codes, scales, w = mo.mxfp4(rand(n, k, seed=2))
    dirty = codes.clone()
    dirty[:, 20:] = 0x77
    args = (x.to(DEV), scales.to(DEV))
    clean = K.mxfp4_linear(args[0], codes.to(DEV), args[1], quantize_input=both)
    assert torch.equal(K.mxfp4_linear(args[0], dirty.to(DEV), args[1], quantize_input=both), clean)
    near(clean, mo.linear(x, w, both=both), k)


def test_mxfp4_linear_non_finite(K):
    """A block with a NaN or an Inf, in x or in the weights, leaves no finite number where it enters and touches nothing else."""
    for m in (4, 200):
        x = rand(m, 96, seed=5)
        w = rand(40, 96, seed=6)
        x[2, 70] = float("nan")
        w[3, 10] = float("inf")
        codes, scales, wv = mo.mxfp4(w)
        for both in (False, True):
            y = K.mxfp4_linear(x.to(DEV), codes.to(DEV), scales.to(DEV), quantize_input=both).cpu()
            ref = mo.linear(x, wv, both=both)
            assert torch.equal(torch.isfinite(y), torch.isfinite(ref))
            fine = torch.isfinite(ref)
            assert rel(y[fine], ref[fine]) < tolerance(torch.float32, 96)


# ---------------------------------------------------------------------------------------- 8-bit checkpoints
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tanh", [False, True])
@pytest.mark.parametrize("m,k,n", LAYERS + [(2000, 130, 140), (5000, 50, 128)])
def test_linear_ckpt8(K, m, k, n, tanh, dtype):
    x = uneven(m, k, dtype, seed=m + k)
    w = rand(k, n, seed=n, scale=(2.0 / (k + n)) ** 0.5, dtype=dtype)
    bias, g = rand(n, seed=2, dtype=dtype), rand(m, n, seed=3, scale=1e-2, dtype=dtype)
    op = K.fused_tanh_linear_ckpt8_autograd if tanh else K.linear_ckpt8_autograd
    for use in (None, bias):
        y_ref, gx_ref, gw_ref, gb_ref = mo.linear_ckpt8(x, w, use, tanh, g)
        leaves = [t.to(DEV).requires_grad_() for t in (x, w) + (() if use is None else (use,))]
        y = op(*leaves)
        near(y, y_ref, k, "y")
        got = torch.autograd.grad(y, leaves, g.to(DEV))
        assert all(t.dtype == dtype for t in got)
        near(got[0], gx_ref, n, "gx")
        near(got[1], gw_ref, m, "gw")
        if use is not None:
            near(got[2], gb_ref, m, "gb")


def test_linear_ckpt8_each_gradient_alone(K):
    x, w, b, g = rand(77, 50, seed=1), rand(50, 33, seed=2), rand(33, seed=3), rand(77, 33, seed=4)
    for op in (K.linear_ckpt8_autograd, K.fused_tanh_linear_ckpt8_autograd):
        full = [t.to(DEV).requires_grad_() for t in (x, w, b)]
        want = torch.autograd.grad(op(*full), full, g.to(DEV))
        for i in range(3):
            leaves = [t.to(DEV).requires_grad_(j == i) for j, t in enumerate((x, w, b))]
            (got,) = torch.autograd.grad(op(*leaves), [leaves[i]], g.to(DEV))
            assert torch.equal(got, want[i])
        assert not op(*[t.to(DEV) for t in (x, w, b)]).requires_grad


def test_no_rows(K):
    w, b = rand(40, 7, seed=1).to(DEV).requires_grad_(), rand(7, seed=2).to(DEV).requires_grad_()
    x = torch.empty(0, 40, device=DEV, requires_grad=True)
    y = K.fused_tanh_linear_ckpt8_autograd(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty(0, 7, device=DEV))
    assert y.shape == (0, 7) and gx.shape == (0, 40) and float(gw.abs().max()) == 0.0 and float(gb.abs().max()) == 0.0
    c, s = K.mxfp4_quantize(w.detach().t().contiguous())
    y = K.mxfp4_linear_autograd(x, c, s, b, "tanh")
    gx, gb = torch.autograd.grad(y, (x, b), torch.empty(0, 7, device=DEV))
    assert y.shape == (0, 7) and gx.shape == (0, 40) and float(gb.abs().max()) == 0.0
