"""Block-scaled layers without a GPU: refusals of the Python and of the C entry points, the oracle's own consistency, and what
the module swaps do to a model's structure."""
import ctypes

import pytest
import torch

from oracle import mx_oracle as mo

FP4 = torch.uint8


def test_oracle_blocks_by_hand():
    x = torch.tensor([[0.3, -0.3, 7.9, 1.0] + [0.0] * 28 + [1e-3]])
    codes, scales, values = mo.mxfp4(x)
    # amax 7.9: E = 2 - 2 = 0, so 0.3 -> 0.5, 7.9 -> 6, 1 -> 1; the short second block: 1e-3 = 1.024 * 2^-10, E = -12
    assert values[0, :4].tolist() == [0.5, -0.5, 6.0, 1.0] and scales.tolist() == [[127, 115]]
    assert codes[0, :2].tolist() == [0x1 | 0x9 << 4, 0x7 | 0x2 << 4] and float(values[0, 32]) == 4 * 2.0 ** -12
    codes, scales, values = mo.mxint8(x)
    assert scales.tolist() == [[129, 117]] and codes[0, :4].tolist() == [5, -5, 126, 16] and codes.shape == (1, 64)
    assert float(values[0, 2]) == 126 / 64 * 4


def test_kept_values_of_fp16_inputs_are_fp16_numbers():
    """What lets a wide fp16 layer hold x8 in one fp16 plane: an fp16 input is a multiple of 2^-24, so that its code is one of 2^-24 / 2^(E-6)
    where that is more than one, and 127 / 64 2^15 is below fp16's largest.  Every magnitude there is, beside every block exponent."""
    bits = torch.arange(1, 0x7c00, dtype=torch.int32).to(torch.int16)
    every = bits.view(torch.float16)                          # ascending: 31743 magnitudes
    for top in range(-24, 16):                                # the exponent of the block's largest
        below = every[every.double() < 2.0 ** (top + 1)]
        below = torch.cat((below, -below, torch.zeros(-2 * below.numel() % 31, dtype=torch.float16))).view(-1, 31)
        x = torch.cat((torch.full((below.shape[0], 1), 2.0 ** top, dtype=torch.float16), below), dim=1)
        values = mo.mxint8(x)[2]
        assert torch.equal(values.half().double(), values)


def test_cpu_tensors_are_refused():
    import flashmd_amd.kernels as K

    x, w, b = torch.zeros(4, 32), torch.zeros(32, 8), torch.zeros(8)
    codes, scales = torch.zeros(8, 16, dtype=FP4), torch.zeros(8, 1, dtype=torch.uint8)
    for f in (lambda: K.mxfp4_quantize(x), lambda: K.mxint8_quantize(x), lambda: K.mxfp4_dequantize(codes, scales, 32),
              lambda: K.mxint8_dequantize(torch.zeros(8, 32, dtype=torch.int8), scales, 32), lambda: K.mxfp4_linear(x, codes, scales),
              lambda: K.mxfp4_linear_autograd(x, codes, scales, b), lambda: K.linear_ckpt8_autograd(x, w, b),
              lambda: K.fused_tanh_linear_ckpt8_autograd(x, w, b)):
        with pytest.raises(RuntimeError, match="GPU"):
            f()


def test_names_are_public():
    import flashmd_amd.kernels as K

    for name in ("mxfp4_quantize", "mxfp4_dequantize", "mxint8_quantize", "mxint8_dequantize", "mxfp4_linear", "mxfp4_linear_autograd",
                 "linear_ckpt8_autograd", "fused_tanh_linear_ckpt8_autograd"):
        assert name in K.__all__ and callable(getattr(K, name))


def test_c_entries_refuse_bad_arguments():
    """Before anything is launched: sizes, types, null and misaligned pointers (the addresses are never read)."""
    from flashmd_amd import _ffi

    lib = _ffi.lib()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4097)
    BAD, OK = -1, 0
    for f in (lib.fmd_mxfp4_quantize, lib.fmd_mxint8_quantize):
        assert f(p, 3, 4, 32, p, p, None) == BAD and f(p, 0, -1, 32, p, p, None) == BAD and f(p, 0, 4, 0, p, p, None) == BAD
        assert f(None, 0, 4, 32, p, p, None) == BAD and f(odd, 0, 4, 32, p, p, None) == BAD and f(p, 0, 4, 32, odd, p, None) == BAD
        assert f(p, 0, 4, 32, p, None, None) == BAD and f(None, 0, 0, 32, None, None, None) == OK
    for f in (lib.fmd_mxfp4_dequantize, lib.fmd_mxint8_dequantize):
        assert f(p, p, 4, 32, p, 5, None) == BAD and f(p, p, 4, 0, p, 0, None) == BAD and f(p, None, 4, 32, p, 0, None) == BAD
        assert f(p, p, 4, 32, odd, 0, None) == BAD and f(None, None, 0, 32, None, 0, None) == OK

    ws = lib.fmd_mxfp4_linear_workspace_bytes
    assert ws(9, 4, 8, 32, 0) == BAD and ws(0, 4, 0, 32, 0) == BAD and ws(0, -4, 8, 32, 0) == BAD and ws(0, 4, 8, 1 << 25, 0) == BAD
    assert ws(0, 0, 8, 32, 0) == 0 and ws(0, 1000, 128, 128, 1) == 0 and ws(2, 64, 4096, 4096, 0) == 0 and ws(2, 65, 4096, 4096, 0) > 0
    f = lib.fmd_mxfp4_linear
    assert f(None, 0, p, p, None, p, None, 4, 8, 32, 0, 0, None, None) == BAD and f(odd, 0, p, p, None, p, None, 4, 8, 32, 0, 0, None, None) == BAD
    assert f(p, 0, odd, p, None, p, None, 4, 8, 32, 0, 0, None, None) == BAD and f(p, 0, p, None, None, p, None, 4, 8, 32, 0, 0, None, None) == BAD
    assert f(p, 0, p, p, None, p, p, 4, 8, 32, 0, 0, None, None) == BAD                       # dact without tanh
    assert f(p, 0, p, p, None, p, None, 1000, 8, 300, 0, 0, None, None) == BAD                # a workspace is needed
    assert f(p, 0, p, p, None, p, None, 1000, 8, 300, 0, 0, odd, None) == BAD
    assert f(p, 0, p, p, None, p, None, 1 << 31, 8, 300, 0, 1, p, None) == BAD                # rows of a 4-bit x are counted in 32 bits
    assert f(None, 0, None, None, None, None, None, 0, 8, 32, 0, 0, None, None) == OK

    f = lib.fmd_mxfp4_linear_bwd
    assert f(p, 0, None, 3, p, p, p, p, 4, 8, 32, p, None) == BAD and f(p, 0, None, 1, p, p, p, p, 4, 8, 32, p, None) == BAD
    assert f(p, 0, p, 2, p, p, p, p, 4, 8, 32, p, None) == BAD and f(p, 1, p, 1, p, p, p, p, 4, 8, 32, p, None) == BAD
    assert f(None, 0, None, 0, p, p, p, p, 4, 8, 32, p, None) == BAD and f(p, 0, None, 0, None, p, p, p, 4, 8, 32, p, None) == BAD
    assert f(p, 0, None, 0, p, p, p, None, 1000, 8, 300, None, None) == BAD
    assert f(p, 0, None, 0, p, p, None, None, 4, 8, 32, None, None) == OK                     # nothing is wanted

    f = lib.fmd_linear_ckpt8
    assert f(p, 0, p, None, p, p, None, 4, 8, 32, 0, None, None) == BAD                       # codes without scales
    assert f(p, 0, None, None, p, p, p, 4, 8, 32, 0, None, None) == BAD and f(p, 0, p, None, odd, p, p, 4, 8, 32, 0, None, None) == BAD
    assert f(p, 0, p, None, p, p, p, 4, 8, 300, 0, None, None) == BAD and f(None, 0, None, None, None, None, None, 0, 8, 32, 0, None, None) == OK
    f = lib.fmd_linear_ckpt8_bwd
    assert f(p, 0, p, p, p, p, p, p, 0, 8, 32, 0, None, None) == BAD and f(p, 0, None, None, p, None, p, None, 4, 8, 32, 0, p, None) == BAD
    assert f(p, 0, None, None, p, p, None, None, 4, 8, 32, 1, p, None) == BAD                 # tanh' needs the checkpoint
    assert f(p, 0, None, None, None, p, None, None, 4, 8, 32, 0, p, None) == BAD              # gx needs the weight
    assert f(p, 0, p, p, p, None, None, None, 4, 8, 32, 0, None, None) == OK
    assert lib.fmd_linear_ckpt8_bwd_workspace_bytes(0, 0, 8, 32, 0, 1, 1, 1) == 0
    assert lib.fmd_linear_ckpt8_bwd_workspace_bytes(0, 4, 8, -2, 0, 1, 1, 1) == BAD


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are not a GPU's: only where every launch fails")
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_a_failed_launch_is_reported(dtype):
    """Where no kernel can be launched, no path of an entry point may answer that it went well."""
    from flashmd_amd import _ffi

    lib, p, FAILED = _ffi.lib(), ctypes.c_void_p(1 << 20), -2
    for m, n, k in ((40, 64, 64), (40, 300, 300), (5000, 64, 64), (100000, 64, 64), (500, 300, 300), (5000, 300, 300)):
        for both in (0, 1):
            assert lib.fmd_mxfp4_linear(p, dtype, p, p, p, p, None, m, n, k, 0, both, p, None) == FAILED
        for gx, gb in ((p, None), (None, p), (p, p)):
            assert lib.fmd_mxfp4_linear_bwd(p, dtype, None, 0, p, p, gx, gb, m, n, k, p, None) == FAILED
        for tanh in (0, 1):
            assert lib.fmd_linear_ckpt8(p, dtype, p, p, p, p, p, m, n, k, tanh, p, None) == FAILED
            for gx, gw, gb in ((p, None, None), (None, p, None), (None, None, p), (p, p, p)):
                assert lib.fmd_linear_ckpt8_bwd(p, dtype, p, p, p, gx, gw, gb, m, n, k, tanh, p, None) == FAILED
    for f in (lib.fmd_mxfp4_quantize, lib.fmd_mxint8_quantize):
        assert f(p, dtype, 4, 40, p, p, None) == FAILED
    for f in (lib.fmd_mxfp4_dequantize, lib.fmd_mxint8_dequantize):
        assert f(p, p, 4, 40, p, dtype, None) == FAILED


def test_sizes_beyond_the_grids_are_refused():
    """A dimension of a weight past 2^20, rows past 2^34, 4-bit rows past 2^29, or a matrix past 2^38 elements: refused before a
    grid or an index could wrap."""
    from flashmd_amd import _ffi

    lib, p, BAD, top = _ffi.lib(), ctypes.c_void_p(1 << 20), -1, 1 << 20
    for m, n, k in ((4, top + 1, 8), (4, 8, top + 1), ((1 << 34) + 1, 8, 8), (1 << 30, 257, 8), (1 << 30, 8, 257), (4, top, (1 << 18) + 1)):
        assert lib.fmd_mxfp4_linear_workspace_bytes(0, m, n, k, 0) == BAD
        assert lib.fmd_mxfp4_linear(p, 0, p, p, None, p, None, m, n, k, 0, 0, p, None) == BAD
        assert lib.fmd_mxfp4_linear_bwd_workspace_bytes(0, m, n, k, 1, 1) == BAD
        assert lib.fmd_mxfp4_linear_bwd(p, 0, None, 0, p, p, p, p, m, n, k, p, None) == BAD
        assert lib.fmd_linear_ckpt8_workspace_bytes(0, m, n, k) == BAD
        assert lib.fmd_linear_ckpt8(p, 0, p, None, p, p, p, m, n, k, 0, p, None) == BAD
        assert lib.fmd_linear_ckpt8_bwd_workspace_bytes(0, m, n, k, 0, 1, 1, 1) == BAD
        assert lib.fmd_linear_ckpt8_bwd(p, 0, p, p, p, p, p, p, m, n, k, 0, p, None) == BAD
    for n, k in ((8, 8), (8, 300)):
        assert lib.fmd_mxfp4_linear_workspace_bytes(0, (1 << 29) + 1, n, k, 1) == BAD
        assert lib.fmd_mxfp4_linear(p, 0, p, p, None, p, None, (1 << 29) + 1, n, k, 0, 1, p, None) == BAD
    assert lib.fmd_mxfp4_linear_workspace_bytes(0, 65, top, 300, 0) > 0 and lib.fmd_mxfp4_linear_workspace_bytes(0, 1 << 29, 8, 300, 1) > 0


def test_misaligned_results_are_refused():
    from flashmd_amd import _ffi

    lib, p, odd, BAD = _ffi.lib(), ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 2), -1
    for m, n, k in ((4, 8, 32), (5000, 300, 300)):
        assert lib.fmd_mxfp4_linear(p, 1, p, p, None, p, odd, m, n, k, 1, 0, p, None) == BAD     # dact
        assert lib.fmd_linear_ckpt8_bwd(p, 1, p, p, p, None, odd, None, m, n, k, 0, p, None) == BAD  # gw


def test_workspaces_do_not_grow_with_the_rows():
    """Large batches go through the wide path in chunks: what the planes of one take, not of all."""
    from flashmd_amd import _ffi

    lib = _ffi.lib()
    one = lib.fmd_linear_ckpt8_workspace_bytes(0, 1 << 20, 300, 300)
    assert 0 < one < 1 << 29 and lib.fmd_linear_ckpt8_workspace_bytes(0, 1 << 26, 300, 300) <= one + (1 << 20)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("k,n", [(300, 300), (2000, 1000), (8192, 8192), (16384, 16384), (20000, 300)])
def test_workspaces_of_gradients_do_not_grow_with_the_rows(k, n, dtype):
    """The weight gradient's sums over chunks of rows: one chunk's planes (128 MiB, or 1024 rows), four [k, n] matrices in fp32 or 128 MiB
    of smaller ones, and what the weight and the sums of the bias take, whatever the rows."""
    from flashmd_amd import _ffi

    lib, mib = _ffi.lib(), 1 << 20
    for tanh in (0, 1):
        at = [lib.fmd_linear_ckpt8_bwd_workspace_bytes(dtype, m, n, k, tanh, 1, 1, 1) for m in (1 << 16, 1 << 18, 1 << 20, 1 << 23)]
        planes = max(128 * mib, 1024 * 6 * (k + n + 64))
        assert max(at) <= 2 * planes + max(128 * mib, 4 * 4 * k * n) + 6 * (n + 64) * k + 64 * mib, (tanh, at)
        assert at[3] - at[2] <= mib
    at = [lib.fmd_mxfp4_linear_bwd_workspace_bytes(dtype, m, n, k, 1, 1) for m in (1 << 18, 1 << 20, 1 << 23)]
    assert at[2] - at[1] <= mib and at[2] <= 128 * mib + 1024 * 6 * (n + 64) + 2 * (n + 64) * k + 64 * mib


@pytest.mark.parametrize("op", ["linear_ckpt8_autograd", "fused_tanh_linear_ckpt8_autograd", "mxfp4_linear_autograd", "mxfp4_tanh"])
def test_gradients_are_not_differentiated_again(op, monkeypatch):
    """create_graph=True with a gradient that is a constant (energies summed for forces): a loss of the result may not come back
    without the layer's part, whichever of the layer's inputs, or of what is before them, it is differentiated for.  The graph
    alone is looked at: the kernels are left out."""
    import flashmd_amd.kernels as K
    from flashmd_amd import _ffi, mx

    monkeypatch.setattr(_ffi, "require_gpu", lambda *t: None)
    monkeypatch.setattr(mx, "_launch", lambda *a: None)
    before, x0 = torch.randn(8, 40, requires_grad=True), torch.randn(5, 8, requires_grad=True)
    b = torch.randn(6, requires_grad=True)
    if op.startswith("mxfp4"):
        codes, scales = torch.zeros(6, 32, dtype=FP4), torch.zeros(6, 2, dtype=torch.uint8)
        leaves = [before, x0, b]
        f = lambda x: K.mxfp4_linear_autograd(x, codes, scales, b, "tanh" if op == "mxfp4_tanh" else None)
    else:
        w = torch.randn(40, 6, requires_grad=True)
        leaves = [before, x0, b, w]
        f = lambda x: getattr(K, op)(x, w, b)
    for factor in (1.0, torch.ones(1, requires_grad=True)):
        y = f(x0 @ before)
        forces = torch.autograd.grad((y * factor).sum(), x0, create_graph=True)[0]
        for leaf in leaves:
            with pytest.raises(RuntimeError, match="differentiated again"):
                torch.autograd.grad((forces * forces).sum(), leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            ((forces * forces).sum() + y.sum()).backward(retain_graph=True)
        for g in torch.autograd.grad(y.sum(), leaves, create_graph=True):
            g.mul_(2.0)                                       # theirs to change
        # a loss of the outputs beside them is no second derivative
        assert all(g.shape == t.shape for g, t in zip(torch.autograd.grad(y.sum(), leaves), leaves))


def test_sizes_are_checked_under_python_O():
    """With assert statements dropped: what does not fit is refused before anything is launched (the launch is replaced)."""
    import os
    import subprocess
    import sys

    code = """
import torch
import flashmd_amd.kernels as K
from flashmd_amd import _ffi, mx
assert False, "assertions are on"
_ffi.require_gpu = lambda *t: None
def launched(*a): raise SystemExit("launched " + a[1])
mx._launch = launched
x, w, b = torch.zeros(4, 40), torch.zeros(40, 8), torch.zeros(8)
codes, scales, c8 = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8), torch.zeros(8, 64, dtype=torch.int8)
n = 0
for f in (lambda: K.mxfp4_quantize(x.double()), lambda: K.mxfp4_quantize(x[0]), lambda: K.mxint8_quantize(x.t()), lambda: K.mxfp4_quantize(x[:, :0].contiguous()),
          lambda: K.mxfp4_dequantize(codes, scales, 65), lambda: K.mxfp4_dequantize(codes[:5], scales, 40), lambda: K.mxint8_dequantize(codes, scales, 40),
          lambda: K.mxint8_dequantize(c8, scales[:, :1].contiguous(), 40), lambda: K.mxfp4_dequantize(codes, scales, 40, torch.float64),
          lambda: K.mxfp4_linear(torch.zeros(4, 70), codes, scales), lambda: K.mxfp4_linear(x, codes, scales, b[:7]),
          lambda: K.mxfp4_linear(x, codes, scales, b.half()), lambda: K.mxfp4_linear(x, codes, scales, activation="relu"),
          lambda: K.mxfp4_linear_autograd(x, codes[:0], scales[:0]), lambda: K.linear_ckpt8_autograd(x, w[:39]), lambda: K.linear_ckpt8_autograd(x, w.half()),
          lambda: K.fused_tanh_linear_ckpt8_autograd(x, w, b[:3]), lambda: K.linear_ckpt8_autograd(x, w[:, :0].contiguous())):
    try:
        f()
    except AssertionError as e:
        n += bool(str(e))
print("refused", n)
"""
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=os.path.join(here, "flash-molecular-dynamics_amd"))
    p = subprocess.run([sys.executable, "-O", "-c", code], env=env, capture_output=True, text=True, timeout=110)
    assert p.stdout.strip() == "refused 18", (p.stdout, p.stderr[-500:])


class _Unmoved(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.sum().detach()

    @staticmethod
    def backward(ctx, g):
        return None


@pytest.mark.parametrize("create_graph", [False, True])
def test_an_undefined_gradient_counts_as_zeros(create_graph, monkeypatch):
    """What comes behind a layer may pass it no gradient at all: its own are then those of zeros, in shape and presence."""
    import flashmd_amd.kernels as K
    from flashmd_amd import _ffi, mx

    seen = []
    monkeypatch.setattr(_ffi, "require_gpu", lambda *t: None)
    monkeypatch.setattr(mx, "_launch", lambda device, name, *a: seen.append(name))
    x, w, b = (torch.randn(*s, requires_grad=True) for s in ((5, 40), (40, 6), (6,)))
    codes, scales = torch.zeros(6, 32, dtype=FP4), torch.zeros(6, 2, dtype=torch.uint8)
    for y, leaves, name in ((K.fused_tanh_linear_ckpt8_autograd(x, w, b), (x, w, b), "fmd_linear_ckpt8_bwd"),
                            (K.mxfp4_linear_autograd(x, codes, scales, b, "tanh"), (x, b), "fmd_mxfp4_linear_bwd")):
        got = torch.autograd.grad(_Unmoved.apply(y), leaves, create_graph=create_graph)
        assert seen[-1] == name and all(g.shape == t.shape for g, t in zip(got, leaves))
    y = K.linear_ckpt8_autograd(x, w, b)                      # nor the gradient one of its own
    gx = torch.autograd.grad(y.sum(), x, create_graph=True)[0]
    assert torch.autograd.grad(_Unmoved.apply(gx) + (w * 0.0).sum(), w)[0].shape == w.shape


def _model(activation=None):
    import flashmd_amd.schnet as S

    return S.StandardSchNet(S.GaussianBasis(S.CosineCutoff(0.0, 5.0), 20), S.CosineCutoff(0.0, 5.0), [16, 8], hidden_channels=16,
                            embedding_size=10, num_filters=16, num_interactions=2, activation=activation)


def test_activation_checkpoints_setting():
    import flashmd_amd.schnet as S

    model = _model()
    names = list(model.state_dict())
    with pytest.raises(ValueError, match="4 bits"):
        S.set_activation_checkpoints(model, bits=4)
    with pytest.raises(ValueError, match="no MLP"):
        S.set_activation_checkpoints(torch.nn.Linear(2, 2))
    assert S.set_activation_checkpoints(model) is model
    marked = [m for m in model.modules() if isinstance(m, (S.MLP, S.InteractionBlock))]
    assert len(marked) == 5 and all(m.checkpoint_bits == 8 for m in marked) and list(model.state_dict()) == names
    with pytest.raises(RuntimeError, match="GPU"):
        model.output_network(torch.zeros(3, 16))
    S.set_activation_checkpoints(model, bits=None)
    assert all(m.checkpoint_bits is None for m in marked) and model.output_network(torch.zeros(3, 16)).shape == (3, 1)
    other = _model(torch.nn.SiLU())
    with pytest.raises(ValueError, match="tanh"):
        S.set_activation_checkpoints(other)
    assert all(m.checkpoint_bits is None for m in other.modules() if isinstance(m, (S.MLP, S.InteractionBlock)))


def test_activation_checkpoints_are_for_training_alone():
    """In eval() the layers run as they are: on the CPU with plain torch, where the checkpointed ones would refuse."""
    import flashmd_amd.schnet as S

    model, x = _model(), torch.randn(5, 16)
    nets = (model.output_network, model.interaction_blocks[0].conv.filter_network)
    want = [net(x if net is model.output_network else x.repeat(1, 2)[:, :20]) for net in nets]
    S.set_activation_checkpoints(model).eval()
    got = [net(x if net is model.output_network else x.repeat(1, 2)[:, :20]) for net in nets]
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    model.train()
    with pytest.raises(RuntimeError, match="GPU"):
        model.output_network(x)


def test_modules_pickled_before_the_setting_existed():
    """A whole module from an older pickle has no ``checkpoint_bits`` of its own: it runs as it did, and takes the setting."""
    import io

    import flashmd_amd.schnet as S

    model = _model().eval()
    for m in model.modules():
        m.__dict__.pop("checkpoint_bits", None)               # what an older version wrote
    f = io.BytesIO()
    torch.save(model, f)
    f.seek(0)
    old = torch.load(f, weights_only=False)
    x = torch.randn(3, 16)
    assert torch.equal(old.output_network(x), model.output_network(x))
    S.set_activation_checkpoints(old)
    assert sum(m.checkpoint_bits == 8 for m in old.modules() if isinstance(m, (S.MLP, S.InteractionBlock))) == 5
    assert S.MLP.checkpoint_bits is None and S.InteractionBlock.checkpoint_bits is None


def test_mxfp4_swap_refusals():
    from flashmd_amd.mxfp4 import MXFP4MLP, apply_mxfp4_to_model

    model = _model()
    with pytest.raises(RuntimeError, match="GPU"):
        apply_mxfp4_to_model(model)
    assert hasattr(model.output_network, "layers")           # nothing was swapped
    with pytest.raises(RuntimeError, match="No filter networks"):
        apply_mxfp4_to_model(torch.nn.Linear(2, 2))
    with pytest.raises(ValueError, match="tanh"):
        MXFP4MLP.from_mlp(_model(torch.nn.SiLU()).output_network)
    with pytest.raises(RuntimeError, match="GPU"):
        MXFP4MLP()(torch.zeros(2, 3))
