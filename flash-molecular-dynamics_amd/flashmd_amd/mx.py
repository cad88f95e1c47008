"""Linear layers on block-scaled numbers: 32 columns of a row share a power of two (formats: include/flashmd_hip.h).

  mxfp4_quantize / mxfp4_dequantize          4-bit blocks (e2m1 elements)
  mxint8_quantize / mxint8_dequantize        8-bit blocks
  mxfp4_linear[_autograd]                    y = f(x W^T + b) with W -- and, if asked for, x -- in 4-bit blocks
  linear_ckpt8_autograd                      y = x W + b          } for training: the backward pass has x in 8-bit blocks
  fused_tanh_linear_ckpt8_autograd           y = tanh(x) W + b    } instead of the tensor itself

Not part of the reference's surface (its narrowest format is fp16, reference models/gptq.py); conventions are those of
``flashmd_amd.kernels``: contiguous GPU tensors, HIP kernels on torch's current stream, fresh outputs, no CPU fallback.
Dense tensors are float32, float16 or bfloat16, one type within a call.  Sums are held in float32 and results rounded once; a 16-bit
layer with a side beyond 256 also rounds what it computes for a product (tanh of its input, a gradient times tanh') to 16 bits, as
torch's own 16-bit operations do.  The gradients are not differentiable again: what tries,
such as a loss on forces taken with ``create_graph=True``, gets a RuntimeError.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _ffi

__all__ = ["mxfp4_quantize", "mxfp4_dequantize", "mxint8_quantize", "mxint8_dequantize", "mxfp4_linear",
           "mxfp4_linear_autograd", "linear_ckpt8_autograd", "fused_tanh_linear_ckpt8_autograd"]

BLOCK = 32
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # FMD_F32, FMD_F16, FMD_BF16
AUX_NONE, AUX_Y, AUX_DACT = 0, 1, 2


def blocks(k: int) -> int:
    return (k + BLOCK - 1) // BLOCK


def _aligned(t: torch.Tensor) -> torch.Tensor:
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _dense(x: torch.Tensor, what: str = "x") -> int:
    """Checks a dense matrix; its type's number."""
    _ffi.require_gpu(x)
    if x.dim() != 2:
        raise AssertionError(f"{what} must be a matrix, got {x.dim()} dimensions")
    if x.dtype not in DTYPES:
        raise AssertionError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    if not x.is_contiguous():
        raise AssertionError(f"{what} must be contiguous")
    return DTYPES[x.dtype]


def _blocked(codes: torch.Tensor, scales: torch.Tensor, k: int, per_block: int, dtype: torch.dtype):
    _ffi.require_gpu(codes, scales)
    if codes.dtype != dtype or scales.dtype != torch.uint8:
        raise AssertionError(f"codes must be {dtype} and scales uint8")
    if codes.dim() != 2 or scales.dim() != 2 or not codes.is_contiguous() or not scales.is_contiguous():
        raise AssertionError("codes and scales must be contiguous matrices")
    if k < 1 or codes.shape != (scales.shape[0], per_block * blocks(k)) or scales.shape[1] != blocks(k):
        raise AssertionError(f"{k} columns take {blocks(k)} blocks a row: codes {tuple(codes.shape)}, scales {tuple(scales.shape)}")
    if codes.device != scales.device:
        raise AssertionError(f"codes are on {codes.device}, scales on {scales.device}")


def _vector(b: Optional[torch.Tensor], n: int, like: torch.Tensor):
    if b is not None:
        _ffi.require_gpu(b)
        if b.shape != (n,) or b.dtype != like.dtype or not b.is_contiguous() or b.device != like.device:
            raise AssertionError(f"bias must be {n} contiguous {like.dtype} on {like.device}")


# Arguments that do not fit raise AssertionError, like the package's other operators, but from an ``if``: the kernels trust the sizes,
# and ``python -O`` drops assert statements.
#
# A call's host side costs as much as a small layer's kernels, so it is kept short: the library's functions are looked up once,
# workspace sizes once a layer shape, pointers go through ctypes as plain integers.


@functools.lru_cache(maxsize=None)
def _function(name: str):
    return getattr(_ffi.lib(), name)


@functools.lru_cache(maxsize=4096)
def _bytes(name: str, *sizes) -> int:
    nbytes = _function(name)(*sizes)
    if nbytes < 0:
        raise RuntimeError(f"flashmd_amd.{name}: {_ffi.strerror(nbytes)} (sizes {sizes})")
    return nbytes


def _workspace(like: torch.Tensor, name: str, *sizes) -> Optional[torch.Tensor]:
    nbytes = _bytes(name, *sizes)
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


def _at(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _launch(device: torch.device, name: str, *args):
    """The C entry on the tensors' device, whichever is current, on torch's current stream there."""
    if device.index == torch.cuda.current_device():
        rc = _function(name)(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            rc = _function(name)(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc != 0:
        _ffi.check(rc, name)


def _quantize(name: str, x, per_block: int, dtype) -> tuple:
    kind = _dense(x)
    m, k = x.shape
    if k < 1:
        raise AssertionError("no columns to quantise")
    x = _aligned(x.detach())
    codes = torch.empty((m, per_block * blocks(k)), dtype=dtype, device=x.device)
    scales = torch.empty((m, blocks(k)), dtype=torch.uint8, device=x.device)
    _launch(x.device, name, _at(x), kind, m, k, _at(codes), _at(scales))
    return codes, scales


def _dequantize(name: str, codes, scales, num_columns: int, dtype, per_block: int, code_dtype) -> torch.Tensor:
    _blocked(codes, scales, num_columns, per_block, code_dtype)
    if dtype not in DTYPES:
        raise AssertionError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    codes = _aligned(codes)
    out = torch.empty((codes.shape[0], num_columns), dtype=dtype, device=codes.device)
    _launch(codes.device, name, _at(codes), _at(scales), codes.shape[0], num_columns, _at(out), DTYPES[dtype])
    return out


def mxfp4_quantize(x: torch.Tensor) -> tuple:
    """x [M,K] -> (codes uint8 [M, 16 ceil(K/32)], scales uint8 [M, ceil(K/32)])."""
    return _quantize("fmd_mxfp4_quantize", x, BLOCK // 2, torch.uint8)


def mxfp4_dequantize(codes, scales, num_columns: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of 4-bit blocks (exact in float32 and bfloat16; float16 rounds what is beyond its range)."""
    return _dequantize("fmd_mxfp4_dequantize", codes, scales, num_columns, dtype, BLOCK // 2, torch.uint8)


def mxint8_quantize(x: torch.Tensor) -> tuple:
    """x [M,K] -> (codes int8 [M, 32 ceil(K/32)], scales uint8 [M, ceil(K/32)])."""
    return _quantize("fmd_mxint8_quantize", x, BLOCK, torch.int8)


def mxint8_dequantize(codes, scales, num_columns: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of 8-bit blocks (exact in float32 and bfloat16; float16 rounds what is beyond its range)."""
    return _dequantize("fmd_mxint8_dequantize", codes, scales, num_columns, dtype, BLOCK, torch.int8)


class _NotTwice(torch.autograd.Function):
    """Stands between a layer's gradients and everything they depend on, and raises when they are to be differentiated."""

    @staticmethod
    def forward(ctx, anchor, grad_output, *gradients):
        ctx.set_materialize_grads(False)
        return tuple(g.new_empty(0).set_(g) for g in gradients)  # the same memory, but no views, which could not be changed in place

    @staticmethod
    def backward(ctx, *again):
        if all(g is None for g in again):  # reached, but with nothing to pass on
            return (None,) * (2 + len(again))
        raise RuntimeError("flashmd_amd: the gradients of block-scaled layers cannot be differentiated again, so a loss on forces "
                           "cannot be trained through them; use a loss on energies, or the layers they stand for "
                           "(set_activation_checkpoints(model, bits=None))")


def _anchored(ctx, y, need: bool) -> tuple:
    ctx.y_shape = y.shape
    ctx.set_materialize_grads(False)  # the anchor's would be made each time
    return y, y.new_empty(0) if need else None


def _once(backward):
    """For a layer whose forward returns what ``_anchored`` does and saves the anchor, an empty output, last.  Under ``create_graph`` the kernels'
    results would be constants to autograd, and whatever is derived from them would lack their part without a word.  The anchor
    leads to the layer's inputs without keeping them."""

    @functools.wraps(backward)
    def wrapper(ctx, grad_output, _):
        if grad_output is None:  # what comes behind y passed it no gradient
            grad_output = ctx.saved_tensors[-1].new_zeros(ctx.y_shape)
        if not torch.is_grad_enabled():
            return backward(ctx, grad_output)
        with torch.no_grad():
            out = backward(ctx, grad_output)
        there = [i for i, g in enumerate(out) if g is not None]
        found = _NotTwice.apply(ctx.saved_tensors[-1], grad_output, *(out[i] for i in there))
        return tuple(found[there.index(i)] if i in there else None for i in range(len(out)))

    return wrapper


# ==================================================================================================
# y = f(x W^T + b), W in 4-bit blocks
# ==================================================================================================


def _check_linear(x, codes, scales, bias, activation) -> int:
    kind = _dense(x)
    if activation not in (None, "tanh"):
        raise AssertionError(f"activation must be None or 'tanh', got {activation!r}")
    _blocked(codes, scales, x.shape[1], BLOCK // 2, torch.uint8)
    if codes.device != x.device or codes.shape[0] < 1:
        raise AssertionError(f"{codes.shape[0]} rows of codes on {codes.device} for x on {x.device}")
    _vector(bias, codes.shape[0], x)
    return kind


def _linear(x, codes, scales, bias, kind: int, tanh: bool, quantize_input: bool, want_dact: bool) -> tuple:
    m, k = x.shape
    n = codes.shape[0]
    x, codes = _aligned(x), _aligned(codes)
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    dact = torch.empty((m, n), dtype=torch.int16, device=x.device) if want_dact else None
    if m:
        ws = _workspace(x, "fmd_mxfp4_linear_workspace_bytes", kind, m, n, k, quantize_input)
        _launch(x.device, "fmd_mxfp4_linear", _at(x), kind, _at(codes), _at(scales), _at(bias), _at(y), _at(dact), m, n, k, tanh,
                quantize_input, _at(ws))
    return y, dact


def mxfp4_linear(x, codes, scales, bias=None, activation: Optional[str] = None, quantize_input: bool = False) -> torch.Tensor:
    """y [M,N] = f(x W^T + b) for x [M,K] and W [N,K] (nn.Linear's layout) as ``mxfp4_quantize`` returns it; f is tanh or
    nothing.  ``quantize_input``: x, too, is taken in its 4-bit blocks (both operands on the 4-bit matrix instruction);
    without it x is exact and only the weights are narrow."""
    kind = _check_linear(x, codes, scales, bias, activation)
    return _linear(x, codes, scales, bias, kind, activation == "tanh", quantize_input, False)[0]


class MXFP4LinearFunction(torch.autograd.Function):
    """gx = (g f') W, gb = sum g f'.  The codes have no gradient; with ``quantize_input`` the quantisation of x passes the
    gradient on as if it were the identity.  f' comes from y in float32, as 1 - y^2 (off by up to 2^-23, as y is rounded: digits
    are lost near saturation, as everywhere in torch).  In 16 bits 1 - y^2 of the rounded y would be far worse: f' itself is
    kept in 16 bits, computed before y is rounded, within 2^-13 of itself or 2^-27."""

    @staticmethod
    def forward(ctx, x, codes, scales, bias, tanh, quantize_input):
        need = ctx.needs_input_grad[0] or ctx.needs_input_grad[3]
        wide = x.dtype == torch.float32
        y, dact = _linear(x, codes, scales, bias, DTYPES[x.dtype], tanh, quantize_input, tanh and need and not wide)
        ctx.aux_kind = AUX_NONE if not tanh else AUX_Y if wide else AUX_DACT
        ctx.k = x.shape[1]
        y, anchor = _anchored(ctx, y, need)
        ctx.save_for_backward(codes, scales, y if ctx.aux_kind == AUX_Y else dact, anchor)
        return y, anchor

    @staticmethod
    @_once
    def backward(ctx, grad_output):
        codes, scales, aux, _ = ctx.saved_tensors
        want_x, want_b = ctx.needs_input_grad[0], ctx.needs_input_grad[3]
        g = _aligned(grad_output.contiguous())
        m, n = g.shape
        kind = DTYPES[g.dtype]
        gx = torch.empty((m, ctx.k), dtype=g.dtype, device=g.device) if want_x else None
        gb = torch.empty(n, dtype=g.dtype, device=g.device) if want_b else None
        codes = _aligned(codes)
        if m or want_b:
            ws = _workspace(g, "fmd_mxfp4_linear_bwd_workspace_bytes", kind, m, n, ctx.k, want_x, want_b)
            _launch(g.device, "fmd_mxfp4_linear_bwd", _at(g), kind, _at(aux), ctx.aux_kind, _at(codes), _at(scales), _at(gx), _at(gb),
                    m, n, ctx.k, _at(ws))
        return gx, None, None, gb, None, None


def mxfp4_linear_autograd(x, codes, scales, bias=None, activation: Optional[str] = None,
                          quantize_input: bool = False) -> torch.Tensor:
    """``mxfp4_linear`` with gradients of x and bias.  Without ``quantize_input`` the gradient of x is the derivative of what
    was computed, so forces taken through such layers are those of their energy."""
    _check_linear(x, codes, scales, bias, activation)
    return MXFP4LinearFunction.apply(x, codes, scales, bias, activation == "tanh", bool(quantize_input))[0]


# ==================================================================================================
# y = p(x) W + b for training, x kept in 8-bit blocks
# ==================================================================================================


class LinearCkpt8Function(torch.autograd.Function):
    """gx = (g W^T) p'(x8), gw = p(x8)^T g, gb = sum g, x8 the 8-bit blocks of x: 33 bytes for 32 columns are all that is kept
    of x.  The blocks are those of the layer's INPUT, so what the backward pass sees is a function of x's bits and not of the
    last digit of a computed tanh."""

    @staticmethod
    def forward(ctx, x, weight, bias, tanh):
        m, k = x.shape
        n = weight.shape[1]
        kind = DTYPES[x.dtype]
        x, w = _aligned(x), _aligned(weight)
        y = torch.empty((m, n), dtype=x.dtype, device=x.device)
        keep = ctx.needs_input_grad[1] or (tanh and ctx.needs_input_grad[0])
        codes = torch.empty((m, BLOCK * blocks(k)), dtype=torch.int8, device=x.device) if keep else None
        scales = torch.empty((m, blocks(k)), dtype=torch.uint8, device=x.device) if keep else None
        if m:
            ws = _workspace(x, "fmd_linear_ckpt8_workspace_bytes", kind, m, n, k)
            _launch(x.device, "fmd_linear_ckpt8", _at(x), kind, _at(w), _at(bias), _at(y), _at(codes), _at(scales), m, n, k, tanh,
                    _at(ws))
        y, anchor = _anchored(ctx, y, any(ctx.needs_input_grad))
        ctx.save_for_backward(codes, scales, weight, anchor)
        ctx.tanh = tanh
        return y, anchor

    @staticmethod
    @_once
    def backward(ctx, grad_output):
        codes, scales, weight, _ = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        g = _aligned(grad_output.contiguous())
        (m, n), k = g.shape, weight.shape[0]
        new = torch.empty if m else torch.zeros
        gx = new((m, k), dtype=g.dtype, device=g.device) if want_x else None
        gw = new((k, n), dtype=g.dtype, device=g.device) if want_w else None
        gb = new(n, dtype=g.dtype, device=g.device) if want_b else None
        if m:
            kind, w = DTYPES[g.dtype], _aligned(weight)
            ws = _workspace(g, "fmd_linear_ckpt8_bwd_workspace_bytes", kind, m, n, k, ctx.tanh, want_x, want_w, want_b)
            _launch(g.device, "fmd_linear_ckpt8_bwd", _at(g), kind, _at(codes), _at(scales), _at(w), _at(gx), _at(gw), _at(gb), m, n, k,
                    ctx.tanh, _at(ws))
        return gx, gw, gb, None


def _ckpt8(x, weight, bias, tanh: bool) -> torch.Tensor:
    _dense(x)
    _dense(weight, "weight")
    if x.dtype != weight.dtype or x.device != weight.device:
        raise AssertionError("x and weight must have one type and one device")
    if x.shape[1] != weight.shape[0]:
        raise AssertionError(f"Dimension mismatch: x has {x.shape[1]} columns but weight has {weight.shape[0]} rows")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise AssertionError("an empty weight")
    _vector(bias, weight.shape[1], x)
    return LinearCkpt8Function.apply(x, weight, bias, tanh)[0]


def linear_ckpt8_autograd(x, weight, bias=None) -> torch.Tensor:
    """y = x W + b, W [K,N]; the backward pass computes the weight's gradient from x's 8-bit blocks (gx and gb are exact)."""
    return _ckpt8(x, weight, bias, False)


def fused_tanh_linear_ckpt8_autograd(x, weight, bias=None) -> torch.Tensor:
    """y = tanh(x) W + b, W [K,N], as ``fused_tanh_linear_autograd``; the backward pass computes tanh and its derivative from
    x's 8-bit blocks."""
    return _ckpt8(x, weight, bias, True)
