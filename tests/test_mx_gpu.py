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
          (269, 50, 128), (269, 128, 64), (300, 256, 257), (1000, 128, 128), (65, 1000, 300), (2100, 200, 256), (2200, 256, 129)]


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
@pytest.mark.parametrize("m,k,n", LAYERS + [(2000, 130, 140), (5000, 50, 128), (2100, 256, 200), (2500, 170, 256)])
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


# ---------------------------------------------------------------------------------------- refusals and how a call may be made
def test_refusals(K):
    x, w, b = rand(4, 40).to(DEV), rand(40, 8).to(DEV), rand(8).to(DEV)
    codes, scales = K.mxfp4_quantize(w.t().contiguous())
    bad = [lambda: K.mxfp4_quantize(x.double()), lambda: K.mxfp4_quantize(x[0]), lambda: K.mxfp4_quantize(x[:, ::2]),
           lambda: K.mxint8_quantize(x.t()), lambda: K.mxfp4_dequantize(codes, scales, 65), lambda: K.mxfp4_dequantize(codes, scales, 40, torch.int8),
           lambda: K.mxint8_dequantize(codes, scales, 40), lambda: K.mxfp4_linear(x, codes, scales, activation="relu"),
           lambda: K.mxfp4_linear(x[:, :31].contiguous(), codes, scales), lambda: K.mxfp4_linear(x, codes, scales, b.half()),
           lambda: K.mxfp4_linear(x, codes, scales, b[:7]), lambda: K.mxfp4_linear(x, codes.cpu(), scales.cpu()),
           lambda: K.mxfp4_linear(x, codes[:, :16].contiguous(), scales), lambda: K.mxfp4_linear(x, codes.char(), scales),
           lambda: K.linear_ckpt8_autograd(x, w.half()), lambda: K.linear_ckpt8_autograd(x, w.t()), lambda: K.linear_ckpt8_autograd(x, w[:39].contiguous()),
           lambda: K.linear_ckpt8_autograd(x.view(2, 2, 40), w), lambda: K.fused_tanh_linear_ckpt8_autograd(x, w, b[::2]),
           lambda: K.linear_ckpt8_autograd(x[:, :0].contiguous(), w[:0].contiguous())]
    for i, f in enumerate(bad):
        with pytest.raises((AssertionError, RuntimeError)):
            f()
            print("not refused:", i)
    xg = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(K.linear_ckpt8_autograd(xg, w, b).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()                                  # not differentiable again


def test_expanded_gradients_and_backward(K):
    """.sum().backward(): a gradient of stride 0; leaves accumulate over two passes."""
    x, w, b = (t.to(DEV).requires_grad_() for t in (rand(50, 40, seed=1), rand(40, 33, seed=2), rand(33, seed=3)))
    for _ in range(2):
        K.fused_tanh_linear_ckpt8_autograd(x, w, b).sum().backward()
    _, gx, gw, gb = mo.linear_ckpt8(x.detach().cpu(), w.detach().cpu(), b.detach().cpu(), True, torch.full((50, 33), 2.0))
    near(x.grad, gx, 33)
    near(w.grad, gw, 50)
    near(b.grad, gb, 50)


def test_gradients_against_differences(K):
    """Central differences of the operators themselves along a direction, at step d: off by d^2/6 of the third derivative (tanh'''
    is at most 2: d^2/3 of the direction's cube) and by the outputs' rounding over d.  With d = 2^-6 both are below 1e-3 of the
    derivative's scale; the 8-bit checkpoints add at most 2^-7 of a block's largest value to x."""
    m, k, n, d = 64, 50, 40, 2.0 ** -6
    x, w, b, v = rand(m, k, seed=1), rand(n, k, seed=2, scale=0.2), rand(n, seed=3, scale=0.1), rand(m, k, seed=4)
    g = rand(m, n, seed=5)
    codes, scales, _ = mo.mxfp4(w)
    c, s, bg, G = codes.to(DEV), scales.to(DEV), b.to(DEV), g.to(DEV)

    def f(t):
        return float((K.mxfp4_linear(t.to(DEV), c, s, bg, "tanh").double() * G.double()).sum())

    xg = x.to(DEV).requires_grad_()
    (gx,) = torch.autograd.grad(K.mxfp4_linear_autograd(xg, c, s, bg, "tanh"), xg, G)
    diff, grad = (f(x + d * v) - f(x - d * v)) / (2 * d), float((gx.double().cpu() * v.double()).sum())
    scale = float(gx.double().norm()) * float(v.double().norm())
    assert abs(diff - grad) < 1e-3 * scale

    wt = w.t().contiguous()
    for tanh, op in ((False, K.linear_ckpt8_autograd), (True, K.fused_tanh_linear_ckpt8_autograd)):
        leaves = [t.to(DEV).requires_grad_() for t in (x, wt, b)]
        got = torch.autograd.grad(op(*leaves), leaves, G)
        for i, base in enumerate((x, wt, b)):
            u = rand(*base.shape, seed=6 + i)

            def at(sign):
                moved = [t.to(DEV) for t in (x, wt, b)]
                moved[i] = (base + sign * d * u).to(DEV)
                return float((op(*moved).double() * G.double()).sum())

            diff, grad = (at(1) - at(-1)) / (2 * d), float((got[i].double().cpu() * u.double()).sum())
            scale = float(got[i].double().norm()) * float(u.double().norm())
            # a kept value is off by at most 2^-7 of its block's largest: of a gradient's 2-norm at most 2^-7 amax/rms (below 4
            # here), twice over where tanh' and the difference meet
            assert abs(diff - grad) < (1e-3 + (2 * 4 * 2.0 ** -7 if i < 2 else 0.0)) * scale, (tanh, i)


def test_rows_behind_the_last_are_left_alone(K):
    """The C entries write m rows and nothing behind them, in every path that stores rows."""
    from flashmd_amd import _ffi
    from flashmd_amd._ffi import call, ptr, stream

    lib = _ffi.lib()
    for m, k, n in ((1, 50, 33), (33, 128, 128), (37, 64, 20), (45, 40, 64), (20, 300, 70), (100, 300, 131), (300, 130, 64), (70, 200, 250), (3001, 257, 70)):
        x, w, g = rand(m, k, seed=1).to(DEV), rand(k, n, seed=2).to(DEV), rand(m, n, seed=3).to(DEV)
        nb, nbn = (k + 31) // 32, (n + 31) // 32
        wc, wsc = K.mxfp4_quantize(w.t().contiguous())
        more = 40

        def room(*shape, dtype=torch.float32):
            return torch.full(shape, 77, dtype=dtype, device=DEV)

        def behind(t):
            return bool((t[m:] == 77).all())

        for tanh in (0, 1):
            y, c8, s8 = room(m + more, n), room(m + more, 32 * nb, dtype=torch.int8), room(m + more, nb, dtype=torch.uint8)
            ws = torch.empty(max(16, lib.fmd_linear_ckpt8_workspace_bytes(0, m, n, k)), dtype=torch.uint8, device=DEV)
            call("fmd_linear_ckpt8", ptr(x), 0, ptr(w), None, ptr(y), ptr(c8), ptr(s8), m, n, k, tanh, ptr(ws), stream())
            assert behind(y) and behind(c8) and behind(s8)
            gx, gw, gb = room(m + more, k), room(k + more, n), room(n + more)
            ws = torch.empty(max(16, lib.fmd_linear_ckpt8_bwd_workspace_bytes(0, m, n, k, tanh, 1, 1, 1)), dtype=torch.uint8, device=DEV)
            call("fmd_linear_ckpt8_bwd", ptr(g), 0, ptr(c8), ptr(s8), ptr(w), ptr(gx), ptr(gw), ptr(gb), m, n, k, tanh, ptr(ws), stream())
            assert behind(gx) and bool((gw[k:] == 77).all()) and bool((gb[n:] == 77).all())
            for both in (0, 1):
                y = room(m + more, n)
                ws = torch.empty(max(16, lib.fmd_mxfp4_linear_workspace_bytes(0, m, n, k, both)), dtype=torch.uint8, device=DEV)
                call("fmd_mxfp4_linear", ptr(x), 0, ptr(wc), ptr(wsc), None, ptr(y), None, m, n, k, tanh, both, ptr(ws), stream())
                assert behind(y)
            gx, gb = room(m + more, k), room(n + more)
            ws = torch.empty(max(16, lib.fmd_mxfp4_linear_bwd_workspace_bytes(0, m, n, k, 1, 1)), dtype=torch.uint8, device=DEV)
            call("fmd_mxfp4_linear_bwd", ptr(g), 0, ptr(y), tanh, ptr(wc), ptr(wsc), ptr(gx), ptr(gb), m, n, k, ptr(ws), stream())
            assert behind(gx) and bool((gb[n:] == 77).all())
        for q, dq, per, dt in ((K.mxfp4_quantize, "fmd_mxfp4_dequantize", 16, torch.uint8), (K.mxint8_quantize, "fmd_mxint8_dequantize", 32, torch.int8)):
            c, s = q(x)
            out = room(m + more, k)
            call(dq, ptr(c), ptr(s), m, k, ptr(out), 0, stream())
            c2, s2 = room(m + more, per * nb, dtype=dt), room(m + more, nb, dtype=torch.uint8)
            call(dq.replace("dequantize", "quantize"), ptr(x), 0, m, k, ptr(c2), ptr(s2), stream())
            assert behind(out) and behind(c2) and behind(s2) and torch.equal(c2[:m], c) and torch.equal(s2[:m], s)


SIZES = [(77, 50, 128), (300, 128, 128), (40, 300, 130), (300, 300, 130)]


def _step(K, x, w, b, codes, scales, g):
    y = K.fused_tanh_linear_ckpt8_autograd(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    z = K.mxfp4_linear_autograd(x, codes, scales, b, "tanh")
    hx, hb = torch.autograd.grad(z, (x, b), g)
    q = K.mxfp4_linear(x.detach(), codes, scales, quantize_input=True)
    return y.detach(), gx, gw, gb, z.detach(), hx, hb, q


def _inputs(K, m, k, n, seed=0):
    x, w, b, g = rand(m, k, seed=seed), rand(k, n, seed=seed + 1, scale=0.2), rand(n, seed=seed + 2), rand(m, n, seed=seed + 3)
    codes, scales = K.mxfp4_quantize(w.t().contiguous().to(DEV))
    return [t.to(DEV).requires_grad_() for t in (x, w, b)] + [codes, scales, g.to(DEV)]


@pytest.mark.parametrize("m,k,n", SIZES)
def test_repeats_and_other_streams(K, m, k, n):
    """Bitwise the same again, on another stream, and with two streams at work at once (nothing is shared between calls)."""
    one, two = _inputs(K, m, k, n), _inputs(K, m, k, n, seed=10)
    want_one, want_two = _step(K, *one), _step(K, *two)
    assert all(torch.equal(a, b) for a, b in zip(want_one, _step(K, *one)))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            got_one = _step(K, *one)
        with torch.cuda.stream(s2):
            got_two = _step(K, *two)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want_one, got_one)) and all(torch.equal(a, b) for a, b in zip(want_two, got_two))


@pytest.mark.parametrize("m,k,n", SIZES)
def test_captured_and_replayed(K, m, k, n):
    """Forward and backward in one graph; replays with new inputs, eager work between them."""
    ins = _inputs(K, m, k, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(K, *ins)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(K, *ins)
    for i in range(4):
        new = _inputs(K, m, k, n, seed=20 + 10 * i)
        with torch.no_grad():
            for a, b in zip(ins, new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(K, *new)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_offsets_beyond_32_bits(K):
    """2^31 elements and more: the last rows of a tensor whose byte (quantise, layer) and element offsets pass 2^32 and 2^31."""
    m, k = 17_000_003, 128
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV)
    tail = rand(70, k, seed=1, dtype=torch.bfloat16)
    x[-70:] = tail.to(DEV)
    codes, scales = K.mxfp4_quantize(x)
    assert torch.equal(codes[-70:].cpu(), mo.mxfp4(tail)[0]) and torch.equal(scales[-70:].cpu(), mo.mxfp4(tail)[1])
    assert int(codes[:-70].max()) == 0
    values = K.mxfp4_dequantize(codes, scales, k, dtype=torch.bfloat16)
    assert torch.equal(values[-70:].cpu().double(), mo.mxfp4(tail)[2])
    del values, codes, scales
    w, b = rand(k, 8, seed=2, dtype=torch.bfloat16), rand(8, seed=3, dtype=torch.bfloat16)
    xg, wg = x.requires_grad_(), w.to(DEV).requires_grad_()
    y = K.fused_tanh_linear_ckpt8_autograd(xg, wg, b.to(DEV))
    g = torch.zeros(m, 8, dtype=torch.bfloat16, device=DEV)
    gt = rand(70, 8, seed=4, dtype=torch.bfloat16)
    g[-70:] = gt.to(DEV)
    gx, gw = torch.autograd.grad(y, (xg, wg), g)
    y_ref, gx_ref, gw_ref, _ = mo.linear_ckpt8(tail, w, b, True, gt)
    near(y[-70:], y_ref, k)
    near(gx[-70:], gx_ref, 8)
    near(gw, gw_ref, 70)
    wc, wsc, wv = mo.mxfp4(w.t().contiguous().float())
    near(K.mxfp4_linear(x.detach(), wc.to(DEV), wsc.to(DEV))[-70:], mo.linear(tail, wv), k)


@pytest.mark.parametrize("m,k,n", [(70000, 128, 128), (70001, 50, 128), (66000, 100, 30), (300_000, 130, 40), (70016, 64, 64), (70003, 200, 150), (70005, 64, 33), (65600, 33, 128), (66001, 256, 256), (80000, 300, 40)])
def test_many_rows(K, m, k, n):
    """Where the weight gradient sums over slices of the rows, and the wide path goes in chunks; small whole numbers, so that every
    product and sum is exact and the result has to be equal to the last bit."""
    gen = torch.Generator().manual_seed(m)
    x = torch.randint(-2, 3, (m, k), generator=gen).float()
    x[:, 0] = 64.0                                            # with 64 the largest of its block, whole numbers are kept whole
    x[:, 32::32] = 64.0
    w, b = torch.randint(-2, 3, (k, n), generator=gen).float(), torch.randint(-3, 4, (n,), generator=gen).float()
    g = torch.randint(-1, 2, (m, n), generator=gen).float()
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = K.linear_ckpt8_autograd(*leaves)
    gx, gw, gb = torch.autograd.grad(y, leaves, g.to(DEV))
    X, W, G = x.to(DEV).double(), w.to(DEV).double(), g.to(DEV).double()
    assert torch.equal(y.detach().double(), X @ W + b.to(DEV).double()) and torch.equal(gx.double(), G @ W.t().contiguous())
    assert torch.equal(gw.double(), X.t().contiguous() @ G) and torch.equal(gb.double(), G.sum(0))


# ---------------------------------------------------------------------------------------- together, in a model
def _schnet(hidden=32, filters=32, rbf=20):
    import flashmd_amd.schnet as S

    torch.manual_seed(3)
    return S.StandardSchNet(S.GaussianBasis(S.CosineCutoff(0.0, 5.0), rbf), S.CosineCutoff(0.0, 5.0), [32, 16], hidden_channels=hidden,
                            embedding_size=30, num_filters=filters, num_interactions=2)


def _batch(S, dev=DEV, dtype=torch.float32):
    from oracle import schnet_oracle as so

    pos, types, ptr_ = so.synth_batch(3, 37, 5.0)
    return S.Batch(pos.to(dev, dtype), types.to(dev), ptr_.to(dev), max_beads_per_mol=37)


def _plain_run(model, S, params=None):
    """The model in 64 bits on the CPU with plain torch operations; energies, forces, gradients of `params` for sum(energy^2)"""
    from oracle import schnet_oracle as so

    data = _batch(S, "cpu", torch.float64)
    src, dst = so.radius_graph(data.pos.float(), data.ptr, 5.0)
    data.pos.requires_grad_(True)
    x = model.embedding_layer(data.atom_types)
    d = (data.pos[dst] - data.pos[src]).norm(dim=1)
    rbf = model.rbf_layer(d)
    for blk in model.interaction_blocks:
        h = blk.conv.lin1(x)
        wf = blk.conv.filter_network.layers(rbf) * blk.conv.cutoff(d).view(-1, 1)
        h = blk.conv.lin2(torch.zeros_like(h).index_add_(0, dst, h[src] * wf))
        x = x + blk.lin(torch.tanh(h))
    e = torch.zeros(3, dtype=torch.float64).index_add_(0, data.batch, model.output_network.layers(x).flatten())
    forces = -torch.autograd.grad(e.sum(), data.pos, retain_graph=True)[0]
    grads = torch.autograd.grad((e * e).sum(), params) if params else None
    return e.detach(), forces, grads


def test_mxfp4_model_is_the_model_with_rounded_weights():
    """apply_mxfp4_to_model: energies and forces equal those of the same model in 64 bits with the blocks' values as weights (the
    operator path's fp32 budget for them is 1e-5); an engine made before the swap is not used again."""
    import copy

    import flashmd_amd.schnet as S
    from flashmd_amd.mxfp4 import MXFP4MLP, apply_mxfp4_to_model

    model = _schnet().to(DEV).eval()
    plain = copy.deepcopy(model).cpu()
    before = S.GradientsOut(model)(_batch(S)).out["SchNet"]["energy"]     # makes the engine
    apply_mxfp4_to_model(model)
    nets = [(p, q) for p, q in zip([b.conv.filter_network for b in plain.interaction_blocks] + [plain.output_network],
                                   [b.conv.filter_network for b in model.interaction_blocks] + [model.output_network])]
    with torch.no_grad():
        for p, q in nets:
            assert isinstance(q, MXFP4MLP)
            for i, linear in enumerate(p.layers[0::2]):
                linear.weight.copy_(q.weight(i).cpu())
                assert torch.equal(linear.weight.double(), mo.mxfp4(linear.weight.detach())[2])  # blocks of blocks are themselves
    e_ref, f_ref, _ = _plain_run(plain.double(), S)
    out = S.GradientsOut(model)(_batch(S)).out["SchNet"]
    assert not torch.equal(out["energy"].detach(), before.detach())
    assert rel(out["energy"], e_ref) < 1e-5 and rel(out["forces"], f_ref) < 1e-5
    # a copy with narrow activations, too, runs and stays finite
    narrow = _schnet().to(DEV).eval()
    apply_mxfp4_to_model(narrow, quantize_activations=True)
    out = S.GradientsOut(narrow)(_batch(S)).out["SchNet"]
    assert bool(torch.isfinite(out["energy"]).all()) and bool(torch.isfinite(out["forces"]).all())


def test_training_step_with_activation_checkpoints():
    """set_activation_checkpoints: energies as without; the parameters' gradients of a loss of the energies against 64 bits.  A
    kept value is off by at most 2^-7 of its block's largest, uniformly: 2^-7 / sqrt(3) of amax in the root mean square, with
    amax at most 4 times the block's rms about 2% of x, and that much of a gradient that is linear in it; a chain of five
    such layers at most 5 times that."""
    import copy

    import flashmd_amd.schnet as S

    model = _schnet().to(DEV).train()
    plain = copy.deepcopy(model).cpu().double()
    names = [n for n, p in model.named_parameters()]
    e_ref, _, want = _plain_run(plain, S, list(plain.parameters()))

    def step():
        e = model(_batch(S)).out["SchNet"]["energy"]
        return e.detach(), torch.autograd.grad((e * e).sum(), list(model.parameters()))

    e0, exact = step()
    S.set_activation_checkpoints(model)
    e8, got = step()
    S.set_activation_checkpoints(model, None)
    assert rel(e0, e_ref) < 1e-5 and rel(e8, e_ref) < 1e-5
    off = {n: rel(g, w) for n, g, w in zip(names, got, want)}
    assert max(off.values()) < 0.1, off
    assert max(rel(g, w) for g, w in zip(exact, want)) < 1e-4
    assert any(v > 1e-4 for v in off.values())               # the checkpoints were used
    e1, again = step()
    assert torch.equal(e1, e0) and all(rel(a, b) < 1e-5 for a, b in zip(again, exact))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k,n", [(50, 128), (64, 64), (33, 127), (7, 30)])
@pytest.mark.parametrize("tanh", [False, True])
def test_both_gradients_of_many_rows(K, k, n, tanh, dtype):
    """Many rows of a narrow layer, against 64 bits on the GPU; gx is bit for bit the same when it is asked for alone.  In fp16 a few of the uneven values are beyond its range: what
    comes of them is not finite where the reference is not, and everything else is as near as ever."""
    m = 66_005
    g = rand(m, n, seed=1, scale=1e-2, dtype=dtype).to(DEV)
    x, w, b = uneven(m, k, dtype, seed=2).to(DEV), rand(k, n, seed=3, scale=0.2, dtype=dtype).to(DEV), rand(n, seed=4, dtype=dtype).to(DEV)
    op = K.fused_tanh_linear_ckpt8_autograd if tanh else K.linear_ckpt8_autograd
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = op(*leaves)
    gx, gw, gb = torch.autograd.grad(y, leaves, g)
    kept = K.mxint8_dequantize(*K.mxint8_quantize(x), k).double()
    G, W = g.double(), w.double()
    p = torch.tanh if tanh else (lambda t: t)

    def finite_near(got, want, terms):
        fine = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), fine)
        near(got[fine], want[fine], terms)

    finite_near(y, p(x.double()) @ W + b.double(), k)
    finite_near(gx, (G @ W.t().contiguous()) * ((1 - torch.tanh(kept) ** 2) if tanh else 1.0), n)
    finite_near(gw, p(kept).t().contiguous() @ G, m)
    finite_near(gb, G.sum(0), m)
    (alone,) = torch.autograd.grad(op(leaves[0], w, b), leaves[:1], g)
    assert torch.equal(torch.nan_to_num(alone), torch.nan_to_num(gx))


def near_where_finite(got, want, terms):
    """An uneven value may be beyond fp16: its block stands for NaN, and what comes of it is not finite in the reference either."""
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got).cpu(), fine)
    near(got.cpu()[fine], want[fine], terms)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tanh", [False, True])
@pytest.mark.parametrize("m,k,n", [(512, 128, 128), (513, 128, 128), (700, 33, 65), (1000, 64, 50), (1025, 7, 30), (500, 300, 300), (513, 300, 257),
                                   (900, 1000, 40), (600, 257, 1), (5000, 300, 300), (6000, 301, 299), (12000, 299, 150), (512, 1024, 1024),
                                   (513, 1024, 1024)])
def test_gradient_of_middling_rows(K, m, k, n, tanh, dtype):
    """Both sides of where the weight gradient takes its rows in parts, and of where it leaves the tiles for the general product."""
    x, w = uneven(m, k, dtype, seed=m + n), rand(k, n, seed=n, scale=(2.0 / (k + n)) ** 0.5, dtype=dtype)
    bias, g = rand(n, seed=2, dtype=dtype), rand(m, n, seed=3, scale=1e-2, dtype=dtype)
    _, _, gw_ref, gb_ref = mo.linear_ckpt8(x, w, bias, tanh, g)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, bias)]
    y = (K.fused_tanh_linear_ckpt8_autograd if tanh else K.linear_ckpt8_autograd)(*leaves)
    gw, gb = torch.autograd.grad(y, leaves[1:], g.to(DEV))
    near_where_finite(gw, gw_ref, m)
    near_where_finite(gb, gb_ref, m)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(98304, 64, 33), (98305, 64, 33), (98305, 50, 128), (98320, 64, 64), (98305, 128, 128), (100001, 33, 127),
                                   (98311, 200, 150), (98310, 129, 30), (98305, 7, 200), (99000, 256, 256)])
def test_gradient_of_many_rows(K, m, k, n, dtype):
    """Both sides of where a narrow layer's weight gradient leaves the tiles; against the oracle, and the same bits twice."""
    x, w = uneven(m, k, dtype, seed=k), rand(k, n, seed=n, scale=(2.0 / (k + n)) ** 0.5, dtype=dtype)
    bias, g = rand(n, seed=2, dtype=dtype), rand(m, n, seed=3, scale=1e-2, dtype=dtype)
    _, _, gw_ref, gb_ref = mo.linear_ckpt8(x, w, bias, True, g)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, bias)]
    first = torch.autograd.grad(K.fused_tanh_linear_ckpt8_autograd(*leaves), leaves[1:], g.to(DEV))
    near_where_finite(first[0], gw_ref, m)
    near_where_finite(first[1], gb_ref, m)
    again = torch.autograd.grad(K.fused_tanh_linear_ckpt8_autograd(*leaves), leaves[1:], g.to(DEV))
    assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(first, again))


@pytest.mark.parametrize("m,k,n", [(98400, 50, 128), (98400, 130, 64), (700, 300, 300)])
def test_streams_and_graphs_beside_the_boundaries(K, m, k, n):
    """The weight gradient over parts of many rows, and the tiles of a wide layer, repeated, on two streams and in a graph."""
    test_repeats_and_other_streams(K, m, k, n)
    test_captured_and_replayed(K, m, k, n)


def test_forces_of_an_evaluation_do_not_go_through_checkpoints(monkeypatch):
    """Operator path, eval(): energies and forces with the setting on are those without it, and the 64-bit model's within the operator
    path's fp32 budget of 1e-5; through 8-bit values they are off by about 1e-2."""
    import copy

    import flashmd_amd.schnet as S

    monkeypatch.setattr(S, "USE_FUSED_ENGINE", False)
    model = _schnet().to(DEV).eval()
    _, f_ref, _ = _plain_run(copy.deepcopy(model).cpu().double(), S)
    want = S.GradientsOut(model)(_batch(S)).out["SchNet"]
    got = S.GradientsOut(S.set_activation_checkpoints(model)).eval()(_batch(S)).out["SchNet"]
    assert rel(got["forces"], f_ref) < 1e-5
    assert rel(got["energy"], want["energy"]) < 1e-5 and rel(got["forces"], want["forces"]) < 1e-5
    model.train()                                             # and in training they do
    data = _batch(S)
    data.pos.requires_grad_(True)
    rounded = -torch.autograd.grad(model(data).out["SchNet"]["energy"].sum(), data.pos)[0]
    assert rel(rounded, f_ref) > 1e-4


def test_a_loss_on_forces_is_refused_with_checkpoints(monkeypatch):
    """GradientsOut in training keeps the graph of the forces.  A loss on energies beside them has the gradients of the bare model's; one
    on forces, which the PyTorch path can differentiate, raises instead of leaving the layers' part out."""
    import flashmd_amd.schnet as S

    for gate, off in (("USE_TRITON_MESSAGE_PASSING", False), ("USE_FUSED_RBF", "0"), ("USE_FUSED_TANH_LINEAR", False), ("USE_CSR", False),
                      ("USE_SRC_CSR_GRAD_X", False), ("USE_FUSED_ENGINE", False)):
        monkeypatch.setattr(S, gate, off)
    model = _schnet().to(DEV).train()
    (S.GradientsOut(model).train()(_batch(S)).out["SchNet"]["forces"] ** 2).sum().backward()
    S.set_activation_checkpoints(model)
    params = list(model.parameters())
    e = model(_batch(S)).out["SchNet"]["energy"]
    want = torch.autograd.grad((e * e).sum(), params)
    out = S.GradientsOut(model).train()(_batch(S)).out["SchNet"]
    with pytest.raises(RuntimeError, match="differentiated again"):
        (out["forces"] ** 2).sum().backward(retain_graph=True)
    got = torch.autograd.grad((out["energy"] ** 2).sum(), params)
    assert all(rel(a, b) < 1e-5 for a, b in zip(got, want))


@pytest.mark.parametrize("dtype,m,k,n", [(torch.float32, 60_000, 2000, 1000), (torch.float32, 26_000, 4200, 2100), (torch.bfloat16, 36_003, 6000, 2999),
                                         (torch.float16, 36_001, 6000, 2999)])
def test_weight_gradient_over_many_chunks(K, dtype, m, k, n):
    """More chunks of rows than sums that are held at once, in parts and whole, the last chunk short.  Small whole numbers: sums are exact
    in fp32 (below 2^24), so every result has to be the exact one rounded once."""
    gen = torch.Generator(device=DEV).manual_seed(m)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=gen, device=DEV).to(dtype)

    x, w, b, g = whole(-2, 3, m, k), whole(-2, 3, k, n), whole(-3, 4, n), whole(-1, 2, m, n)
    x[:, 0::32] = 64.0                                        # with 64 the largest of its block, whole numbers are kept whole
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = K.linear_ckpt8_autograd(*leaves)
    gx, gw, gb = torch.autograd.grad(y, leaves, g)
    with torch.no_grad():
        X, W, G = x.double(), w.double(), g.double()
        assert torch.equal(y, (X @ W + b.double()).to(dtype)) and torch.equal(gx, (G @ W.t().contiguous()).to(dtype))
        assert torch.equal(gw, (X.t().contiguous() @ G).to(dtype)) and torch.equal(gb, G.sum(0).to(dtype))


@pytest.mark.parametrize("dtype,wide", [(torch.float32, 20_000), (torch.float16, 60_000), (torch.bfloat16, 60_000)])
@pytest.mark.parametrize("tanh", [False, True])
def test_checkpointed_layer_across_a_chunk(K, dtype, wide, tanh):
    """Chunks of 1024 rows and a short one of 76: the forward pass's planes and checkpoint (many inputs), the gradient of x with tanh' of the
    checkpoint in its epilogue (many outputs).  The rows behind the first chunk are compared by themselves, too."""
    m, c = 1100, 1024
    for k, n in ((wide, 260), (260, wide)):
        x, w = uneven(m, k, dtype, seed=1), rand(k, n, seed=2, scale=(2.0 / (k + n)) ** 0.5, dtype=dtype)
        x = torch.where(torch.isfinite(x), x, torch.zeros((), dtype=dtype))
        bias, g = rand(n, seed=3, dtype=dtype), rand(m, n, seed=4, scale=1e-2, dtype=dtype)
        leaves = [t.to(DEV).requires_grad_() for t in (x, w, bias)]
        y = (K.fused_tanh_linear_ckpt8_autograd if tanh else K.linear_ckpt8_autograd)(*leaves)
        gx, gw, gb = torch.autograd.grad(y, leaves, g.to(DEV))
        kept = K.mxint8_dequantize(*K.mxint8_quantize(x.to(DEV)), k)
        X, W, G, B = (t.to(DEV).double() for t in (x, w, g, bias))
        p = torch.tanh if tanh else (lambda t: t)
        y_ref, gx_ref = p(X) @ W + B, G @ W.t().contiguous()
        if tanh:
            gx_ref = gx_ref / torch.cosh(kept.double()) ** 2
        for rows in (slice(0, m), slice(c, m)):
            near(y[rows], y_ref[rows], k, "y")
            near(gx[rows], gx_ref[rows], n, "gx")
        near(gw, p(kept.double()).t().contiguous() @ G, m, "gw")
        near(gb, G.sum(0), m, "gb")


@pytest.mark.parametrize("dtype,wide", [(torch.float32, 20_000), (torch.float16, 30_000), (torch.bfloat16, 60_000)])
@pytest.mark.parametrize("tanh", [False, True])
def test_four_bit_layer_across_a_chunk(K, dtype, wide, tanh):
    """The same for 4-bit weights: y and the kept derivative of its tanh (many inputs), the gradient through it (many outputs)."""
    m, c = 1100, 1024
    for k, n in ((wide, 260), (260, wide)):
        x, bias, g = rand(m, k, seed=1, dtype=dtype), rand(n, seed=3, dtype=dtype), rand(m, n, seed=4, scale=1e-2, dtype=dtype)
        codes, scales = K.mxfp4_quantize(rand(n, k, seed=2, scale=(1.0 / k) ** 0.5).to(DEV))
        W = K.mxfp4_dequantize(codes, scales, k).double()
        xg, bg = x.to(DEV).requires_grad_(), bias.to(DEV).requires_grad_()
        y = K.mxfp4_linear_autograd(xg, codes, scales, bg, "tanh" if tanh else None)
        gx, gb = torch.autograd.grad(y, (xg, bg), g.to(DEV))
        z = x.to(DEV).double() @ W.t().contiguous() + bias.to(DEV).double()
        G = g.to(DEV).double() / torch.cosh(z) ** 2 if tanh else g.to(DEV).double()
        y_ref, gx_ref = torch.tanh(z) if tanh else z, G @ W
        for rows in (slice(0, m), slice(c, m)):
            near(y[rows], y_ref[rows], k, "y")
            near(gx[rows], gx_ref[rows], n + (k if tanh else 0), "gx")
        near(gb, G.sum(0), m + (k if tanh else 0), "gb")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(5000, 64, 33), (34_432, 20, 7), (2100, 100, 255), (40, 33, 50), (9000, 128, 129)])
def test_products_with_the_derivative_between_lanes(K, dtype, m, k, n):
    """g f' of rows that no 16-byte piece divides goes through LDS word by word, and is read back by other lanes as rows and as columns.
    With x = 0 and no bias f' is 1: whole numbers give exact gradients, rounded once."""
    gen = torch.Generator().manual_seed(n)
    w, g = torch.randint(-3, 4, (n, k), generator=gen).float(), torch.randint(-2, 3, (m, n), generator=gen).to(dtype)
    w[:, 0::32] = 4.0                                         # blocks whose whole numbers up to 4 are kept whole
    codes, scales, values = mo.mxfp4(w)
    assert torch.equal(values, w.double())
    x, b = torch.zeros(m, k, dtype=dtype, device=DEV).requires_grad_(), torch.zeros(n, dtype=dtype, device=DEV).requires_grad_()
    y = K.mxfp4_linear_autograd(x, codes.to(DEV), scales.to(DEV), b, "tanh")
    gx, gb = torch.autograd.grad(y, (x, b), g.to(DEV))
    assert torch.equal(gx.cpu(), (g.double() @ values).to(dtype)) and torch.equal(gb.cpu(), g.double().sum(0).to(dtype))


def saturated(m, k, dtype, top):
    """values of both signs up to `top`, the larger ones dense"""
    gen = torch.Generator().manual_seed(m)
    x = top * torch.rand(m, k, generator=gen) ** 0.5 * torch.randint(0, 2, (m, k), generator=gen).mul(2).sub(1)
    return x.to(dtype)


def each_near(got, want, top, more=0.0, least=0.0):
    """Element by element.  tanh' = 4 t (1 - t), t = 1 / (e^{2|x|} + 1): 2|x| log2(e) and its constant are rounded (1.5 units in the last
    place of it each way, at most 3 |x| of the result's), the exponential, the reciprocal and three operations by a unit or so each:
    2^-24 (5 |x| + 16); then the type's own half a step, relative or of its smallest number, and what is given as `more` (relative)
    and `least`."""
    t = torch.finfo(got.dtype)
    off = (got.detach().double().cpu() - want).abs()
    tol = (2.0 ** -24 * (5 * top + 16) + more + (t.eps / 2 if got.dtype != torch.float32 else 0.0)) * want.abs() + t.smallest_normal * t.eps / 2 + least
    worst = float((off / tol).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(40, 64), (40, 50), (3000, 64), (100, 300), (300, 1030)])
def test_derivative_of_a_saturated_checkpoint(K, dtype, m, k):
    """tanh' of kept values up to 14, element by element: through an identity weight the gradient of x is g tanh'(x8) and nothing else."""
    top = 14.0
    x, w = saturated(m, k, dtype, top), torch.eye(k, dtype=dtype)
    leaf = x.to(DEV).requires_grad_()
    y = K.fused_tanh_linear_ckpt8_autograd(leaf, w.to(DEV))
    (gx,) = torch.autograd.grad(y, leaf, torch.full((m, k), 1024.0, dtype=dtype, device=DEV))
    each_near(gx, 1024.0 / torch.cosh(mo.mxint8(x)[2]) ** 2, top)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(40, 64), (40, 50), (5, 255), (3000, 64), (40, 300), (100, 300), (300, 1030), (6000, 2100)])
def test_derivative_of_a_saturated_four_bit_layer(K, dtype, m, k):
    """f' of sums up to 14 in 16 bits, element by element: through an identity the gradient of x is g f' and nothing else, in every kernel
    that keeps f' (few rows, narrow, wide, the contraction in parts) and in those that read it.  f' is kept within 2^-13 of itself or 2^-27; in
    fp16 the product g f' is cut to two planes of 8 bits, 2^-15 of it at most."""
    top = 14.0
    x = saturated(m, k, dtype, top)
    codes, scales = K.mxfp4_quantize(torch.eye(k, device=DEV))
    leaf, b = x.to(DEV).requires_grad_(), torch.zeros(k, dtype=dtype, device=DEV).requires_grad_()
    y = K.mxfp4_linear_autograd(leaf, codes, scales, b, "tanh")
    gx, gb = torch.autograd.grad(y, (leaf, b), torch.full((m, k), 1024.0, dtype=dtype, device=DEV))
    want = 1024.0 / torch.cosh(x.double()) ** 2
    each_near(y, torch.tanh(x.double()), top)
    planes = 2.0 ** -15 if dtype == torch.float16 else 0.0
    small = want < 1024.0 * 2.0 ** -14
    each_near(gx[~small], want[~small], top, planes + 2.0 ** -13)
    each_near(gx[small], want[small], top, planes, 1024.0 * 2.0 ** -27)
    near(gb, want.sum(0), m)


def test_kept_derivatives_that_are_exact_or_not_numbers(K):
    """f' of 0 is 1 and of an Inf 0, exactly; of a NaN it is one, in every kernel that keeps or reads it."""
    for dtype in (torch.float16, torch.bfloat16):
        for m, k in ((40, 64), (40, 50), (40, 300), (100, 300), (300, 1030)):
            x = torch.zeros(m, k, dtype=dtype)
            codes, scales = K.mxfp4_quantize(torch.eye(k, device=DEV))
            bias = torch.zeros(k, dtype=dtype)
            bias[1], bias[3], bias[k - 1] = float("inf"), float("nan"), -float("inf")
            leaf, b = x.to(DEV).requires_grad_(), bias.to(DEV).requires_grad_()
            y = K.mxfp4_linear_autograd(leaf, codes, scales, b, "tanh")
            gb, = torch.autograd.grad(y, b, torch.full((m, k), 3.0, dtype=dtype, device=DEV), retain_graph=True)
            want = torch.full((k,), 3.0 * m, dtype=torch.float64)
            want[1], want[3], want[k - 1] = 0.0, float("nan"), 0.0
            assert torch.equal(torch.nan_to_num(gb.double().cpu(), nan=-1.0), torch.nan_to_num(want.to(dtype).double(), nan=-1.0))
            gx, = torch.autograd.grad(y, leaf, torch.full((m, k), 3.0, dtype=dtype, device=DEV))
            assert bool(torch.isnan(gx).all())                # every product has the NaN among its terms, times the identity's zeros


@pytest.mark.parametrize("m,k,n", [(269, 128, 128), (3000, 50, 128), (66_005, 57, 131), (99_000, 128, 100), (400, 300, 300), (5, 7, 200)])
def test_computed_operands_of_narrow_bf16_layers_are_not_rounded(K, m, k, n):
    """tanh(x), tanh(x8) and g f' enter their products in two planes, within 2^-15 of themselves (g f' within 2^-13, as f' is kept), so that
    nearly every result is the exact one rounded once.  A result that is off by e of the results' root mean square R before it is rounded
    rounds otherwise with a chance of about 2^7.5 e R / |v|, for normal v 0.8 r (1 + ln 1/r) on average, r = 2^7.5 e: 4 % for e = 2^-14.3
    (2^-13 in the root mean square), but 50 % for operands rounded to bf16 (e = 2^-9.3)."""
    def otherwise(got, want):
        return float((got.detach() != want.to(torch.bfloat16)).double().mean())

    x, w = rand(m, k, seed=1), rand(k, n, seed=2, scale=(2.0 / (k + n)) ** 0.5, dtype=torch.bfloat16)
    x, g = x.bfloat16(), rand(m, n, seed=3, scale=1e-2, dtype=torch.bfloat16)
    most = 0.12
    leaves = [t.to(DEV).requires_grad_() for t in (x, w)]
    y = K.fused_tanh_linear_ckpt8_autograd(*leaves)
    gw = torch.autograd.grad(y, leaves[1], g.to(DEV))[0]
    X, W, G = x.to(DEV).double(), w.to(DEV).double(), g.to(DEV).double()
    kept = K.mxint8_dequantize(*K.mxint8_quantize(x.to(DEV)), k).double()
    if max(k, n) <= 256:
        assert otherwise(y, torch.tanh(X) @ W) <= most
    assert otherwise(gw, torch.tanh(kept).t().contiguous() @ G) <= most
    codes, scales = K.mxfp4_quantize(w.t().contiguous().to(DEV))
    V = K.mxfp4_dequantize(codes, scales, k).double()
    y = K.mxfp4_linear_autograd(leaves[0], codes, scales, None, "tanh")
    gx = torch.autograd.grad(y, leaves[0], g.to(DEV))[0]
    if max(k, n) <= 256:
        assert otherwise(gx, (G / torch.cosh(X @ V.t().contiguous()) ** 2) @ V) <= most


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 40, 33), (300, 128, 128), (1000, 300, 131), (70_000, 50, 128), (99_001, 256, 255)])
def test_bias_gradient_alone(K, dtype, m, k, n):
    """Whole numbers: the exact sum rounded once, whatever else is asked for."""
    gen = torch.Generator().manual_seed(m)
    g = torch.randint(-2, 3, (m, n), generator=gen).to(dtype).to(DEV)
    x, w, b = rand(m, k, seed=1, dtype=dtype).to(DEV), rand(k, n, seed=2, dtype=dtype).to(DEV), rand(n, seed=3, dtype=dtype).to(DEV)
    want = g.double().sum(0).to(dtype)
    for op in (K.linear_ckpt8_autograd, K.fused_tanh_linear_ckpt8_autograd):
        leaf, weight = b.clone().requires_grad_(), w.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(op(x, w, leaf), leaf, g)[0], want)
        assert torch.equal(torch.autograd.grad(op(x, weight, leaf), (weight, leaf), g)[1], want)
        uneven_g = uneven(m, n, torch.float32, seed=4).clamp(-1e3, 1e3).to(dtype).to(DEV)    # and the same bits alone
        assert torch.equal(torch.autograd.grad(op(x, w, leaf), leaf, uneven_g)[0],
                           torch.autograd.grad(op(x, weight, leaf), (weight, leaf), uneven_g)[1])


class _LayerOnKeptValues(torch.autograd.Function):
    """p(x) W^T + b in 64 bits whose backward pass has the given kept values of x in its place"""

    @staticmethod
    def forward(ctx, x, weight, bias, kept, tanh):
        ctx.save_for_backward(weight, kept)
        ctx.tanh = tanh
        y = (torch.tanh(x) if tanh else x) @ weight.t()
        return y if bias is None else y + bias

    @staticmethod
    def backward(ctx, g):
        weight, kept = ctx.saved_tensors
        p = torch.tanh(kept) if ctx.tanh else kept
        gx = g @ weight
        return gx / torch.cosh(kept) ** 2 if ctx.tanh else gx, g.t() @ p, g.sum(0) if ctx.needs_input_grad[2] else None, None, None


def test_training_step_is_that_of_the_kept_values(monkeypatch):
    """Every parameter's gradient of a loss of energies against the model in 64 bits that has, layer by layer, the very 8-bit values the GPU
    kept: what is left is the operator path's fp32 arithmetic, the 1e-4 that the layers without checkpoints are held to."""
    import copy

    import flashmd_amd.schnet as S
    from oracle import schnet_oracle as so

    model = S.set_activation_checkpoints(_schnet().to(DEV).train())
    plain = copy.deepcopy(model).cpu().double()
    kept = []
    for name in ("linear_ckpt8_autograd", "fused_tanh_linear_ckpt8_autograd"):
        def record(x, weight, bias=None, op=getattr(S.K, name)):
            kept.append((x.detach().cpu().double(), S.K.mxint8_dequantize(*S.K.mxint8_quantize(x), x.shape[1]).cpu().double()))
            return op(x, weight, bias)

        monkeypatch.setattr(S.K, name, record)
    e = model(_batch(S)).out["SchNet"]["energy"]
    got = torch.autograd.grad((e * e).sum(), list(model.parameters()))
    monkeypatch.undo()
    assert len(kept) == 2 * 3 + 3

    used = iter(kept)

    def layer(x, linear, tanh):
        seen, values = next(used)
        assert rel(seen, x) < 1e-5                            # the same rows in the same order
        return _LayerOnKeptValues.apply(x, linear.weight, linear.bias, values, tanh)

    def mlp(x, net):
        for i, linear in enumerate(net.layers[0::2]):
            x = layer(x, linear, i > 0)
        return x

    data = _batch(S, "cpu", torch.float64)
    src, dst = so.radius_graph(data.pos.float(), data.ptr, 5.0)
    x = plain.embedding_layer(data.atom_types)
    d = (data.pos[dst] - data.pos[src]).norm(dim=1)
    rbf = plain.rbf_layer(d)
    for blk in plain.interaction_blocks:
        h = blk.conv.lin1(x)
        wf = mlp(rbf, blk.conv.filter_network) * blk.conv.cutoff(d).view(-1, 1)
        h = blk.conv.lin2(torch.zeros_like(h).index_add_(0, dst, h[src] * wf))
        x = x + layer(h, blk.lin, True)
    energy = torch.zeros(3, dtype=torch.float64).index_add_(0, data.batch, mlp(x, plain.output_network).flatten())
    want = torch.autograd.grad((energy * energy).sum(), list(plain.parameters()))
    off = {n: rel(g, w) for (n, _), g, w in zip(model.named_parameters(), got, want)}
    assert rel(e, energy) < 1e-5 and max(off.values()) < 1e-4, off
