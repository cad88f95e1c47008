"""MXFP4 module swap: the filter and output networks with their weights in 4-bit blocks (17 bytes for 32 weights).

The sibling of the W16A16 swap (flashmd_amd.gptq, reference models/gptq.py:374-443) below 16 bits; the reference has no such
mode.  By default only the weights are narrow: activations stay in the model's type, and the forces are the exact gradient of
the energy the swapped model computes.  ``quantize_activations=True`` also takes every layer's input in its 4-bit blocks; the
energy is then a step function of the positions and the forces are those of the straight-through gradient, which no longer
conserve it: for measuring a model, not for running dynamics.  As in W16A16 there is no CPU path.

A swapped model runs on the operator path, not on the fused engine, which holds 32- or 16-bit networks only: energies and forces of 128
molecules of 269 beads in 10.2 ms, against 14.4 ms on that path in fp32 and 1.75 ms on the engine.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .kernels import mxfp4_dequantize, mxfp4_linear_autograd, mxfp4_quantize


class MXFP4MLP(nn.Module):
    """Linear (+tanh) layers of an ``MLP`` (reference models/mlp.py:6-57), tanh after every one but the last; weights as
    ``codes_<i>``, ``scales_<i>`` buffers, biases as parameters."""

    def __init__(self, quantize_activations: bool = False):
        super().__init__()
        self.quantize_activations = bool(quantize_activations)
        self.num_layers = 0
        self.in_features = []

    @classmethod
    def from_mlp(cls, mlp: nn.Module, quantize_activations: bool = False) -> "MXFP4MLP":
        layers = list(mlp.layers)
        linears, between = layers[0::2], layers[1::2]
        if not linears or len(layers) % 2 == 0 or not all(isinstance(m, nn.Linear) for m in linears) \
                or not all(isinstance(m, nn.Tanh) for m in between):
            raise ValueError("MXFP4 needs an MLP of Linear layers with tanh between them")
        if not linears[0].weight.is_cuda:
            raise RuntimeError("MXFP4 quantisation requires the model on the GPU. "
                               "No CPU fallback is provided to prevent silent bugs.")
        q = cls(quantize_activations)
        for i, linear in enumerate(linears):
            codes, scales = mxfp4_quantize(linear.weight.detach().contiguous())
            q.register_buffer(f"codes_{i}", codes)
            q.register_buffer(f"scales_{i}", scales)
            bias = None if linear.bias is None else nn.Parameter(linear.bias.detach().clone(), linear.bias.requires_grad)
            q.register_parameter(f"bias_{i}", bias)
            q.in_features.append(linear.in_features)
        q.num_layers = len(linears)
        return q.train(mlp.training)

    def weight(self, i: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values of layer i's weight, nn.Linear's [out, in]."""
        return mxfp4_dequantize(getattr(self, f"codes_{i}"), getattr(self, f"scales_{i}"), self.in_features[i], dtype)

    def forward(self, x: torch.Tensor, data=None) -> torch.Tensor:
        if not x.is_cuda:
            raise RuntimeError("MXFP4 network requires a GPU input. No CPU fallback is provided to prevent silent bugs.")
        for i in range(self.num_layers):
            x = mxfp4_linear_autograd(x.contiguous(), getattr(self, f"codes_{i}"), getattr(self, f"scales_{i}"),
                                      getattr(self, f"bias_{i}"), activation="tanh" if i + 1 < self.num_layers else None,
                                      quantize_input=self.quantize_activations)
        return x


def apply_mxfp4_to_model(model: nn.Module, quantize_activations: bool = False) -> nn.Module:
    """Swap every ``filter_network`` and ``output_network`` MLP of ``model`` for its MXFP4 twin, in place.  The fused engine
    holds 32- or 16-bit networks only: a swapped model runs on the operator path, and an engine made before is dropped."""
    found = [(module, name) for module in model.modules() for name in ("filter_network", "output_network")
             if hasattr(getattr(module, name, None), "layers")]
    if not any(name == "filter_network" for _, name in found):
        raise RuntimeError("No filter networks found to quantize. "
                           "Ensure the model contains CFConv layers with filter_network MLPs.")
    twins = [MXFP4MLP.from_mlp(getattr(module, name), quantize_activations) for module, name in found]  # all or none
    for (module, name), twin in zip(found, twins):
        setattr(module, name, twin)
    for module in model.modules():
        if hasattr(module, "_engine"):
            module._engine = None
    return model
