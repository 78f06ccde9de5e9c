"""Layers of a trained block on the MI355X kernels (libdmn_hip.so): layer norm and the linear layer with its epilogue.

What the reference builds its blocks from outside the convolutions -- `Residual(PreNorm(fn))`
(diffusion_model_nemo/utils.py:68-93) and the `nn.Linear` / `nn.GELU` pairs of its embedding networks
(diffusion_model_nemo/modules/unet.py:59-66) -- as calls on device tensors with their backward passes. `layer_norm` and
`linear` are differentiable torch functions; `LayerNorm` and `Linear` hold the parameters under torch's names, so
`state_dict`s interchange with `torch.nn`. There is no CPU implementation: a CPU tensor raises. So do dual tensors (forward-mode
derivatives) and `torch.jit.trace`, which see nothing of what the kernels compute.

Results are rounded once, to the input's type; sums, statistics and parameter gradients are formed in float32. The backward
passes are not differentiable themselves. Calls and their backward passes can be captured into a graph; a call that would be
captured while an eager graph over the same leaves, made on another stream, still lives is refused (its backward would end
the process inside torch, `autograd.grad` as well as `backward`). Whether a backward follows cannot be seen from the call: a
forward alone is captured beside such a graph under `torch.no_grad()`.
"""
from typing import Optional

import torch
import torch.nn as nn

from .. import _native as N

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}
EXACT = 16   # DMN_LINEAR_EXACT of include/dmn.h


def _stream(x: torch.Tensor, what: str):
    """Torch's current stream of x's device; the other checks are in csrc/dmn_torch.cpp."""
    if not x.is_cuda:
        raise RuntimeError(f"{what} runs only on MI355X device tensors (no CPU implementation)")
    return torch._C._cuda_getCurrentRawStream(x.get_device())


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of `x` [..., width] (float32, bfloat16 or float16).
    `weight` and `bias` [width] (either may be None) are of x's type or float32, both alike; their gradients come in
    that type. Rows with any stride are read in place for a 2-D `x`; other layouts are copied first. The statistics are
    float32: a row whose squared deviations add up to more than 3.4e38 comes out as zeros times weight plus bias."""
    return N.ops().layer_norm(x, weight, bias, eps, _stream(x, "layer_norm"))


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, rounded_backward: bool = False) -> torch.Tensor:
    """act(x weight^T + bias) + residual in one pass: `x` [..., in], `weight` [out, in], `bias` [out], `residual` [..., out],
    all of one type (float32, bfloat16 or float16); `activation` None, 'relu', 'silu' or 'gelu' (the exact one). The sum in
    front of the activation, the activation and the residual are formed in float32 and rounded once. Rows with any stride
    below 2^20 are read in place for 2-D tensors, other layouts are copied first. `in` and `out` are below 2^20.

    For the backward with an activation the value z in front of it is kept in float32, and dz = dy act'(z) enters the products
    of a 16-bit type in two parts, so the gradients too are rounded once. `rounded_backward=True` keeps z and dz in the type, as
    a composition of 16-bit layers does: a 16-bit z, half of the backward's matrix work, errors of dx and dweight sqrt 2
    larger. It changes nothing for float32 or without an activation."""
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    return N.ops().linear(x, weight, bias, code if rounded_backward else code | EXACT, residual, _stream(x, "linear"))


class LayerNorm(nn.Module):
    """`layer_norm` over the last axis with parameters `weight` (ones) and `bias` (zeros), as torch.nn.LayerNorm(dim)."""

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None, dtype=None):
        super().__init__()
        if dim < 1:
            raise ValueError("dim must be at least 1")
        self.dim, self.eps = int(dim), float(eps)
        kw = {"device": device, "dtype": dtype}
        self.weight = nn.Parameter(torch.ones(dim, **kw)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(dim, **kw)) if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.dim:
            raise ValueError(f"expected a last axis of {self.dim}, got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)


class Linear(nn.Linear):
    """torch.nn.Linear (its parameters, initialisation and state_dict) with an activation and a residual in its epilogue:
    `Linear(in, out, activation='gelu')(x)`, `Linear(in, out)(x, residual=x0)`. `rounded_backward` as in `linear`."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: Optional[str] = None, device=None,
                 dtype=None, rounded_backward: bool = False):
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        self.activation, self.rounded_backward = activation, bool(rounded_backward)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return linear(x, self.weight, self.bias, self.activation, residual, self.rounded_backward)
