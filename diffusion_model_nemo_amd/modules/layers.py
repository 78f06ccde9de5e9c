"""Layers of a trained block on the MI355X kernels (libdmn_hip.so): layer norm and the linear layer with its epilogue.

What the reference builds its blocks from outside the convolutions -- `Residual(PreNorm(fn))`
(diffusion_model_nemo/utils.py:68-93) and the `nn.Linear` / `nn.GELU` pairs of its embedding networks
(diffusion_model_nemo/modules/unet.py:55-61) -- as calls on device tensors with their backward passes. `layer_norm` and
`linear` are differentiable torch functions; `LayerNorm` and `Linear` hold the parameters under torch's names, so
`state_dict`s interchange with `torch.nn`. There is no CPU implementation: a CPU tensor raises.

Results are rounded once, to the input's type; sums, statistics and parameter gradients are formed in float32. The backward
passes are not differentiable themselves. Calls can be captured into a graph; when a BACKWARD is captured, torch asks that no
eager graph over the same leaves is still alive (capture after warm-up on the capturing stream, as `torch.cuda.graphs`
describes).
"""
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _native as N


def _check_tensor(t: torch.Tensor, what: str):
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs only on MI355X device tensors (no CPU implementation)")
    if t.dtype not in N.DTYPE_CODES:
        raise ValueError(f"{what}: dtype must be float32, bfloat16 or float16, got {t.dtype}")


def _check_param(p: Optional[torch.Tensor], name: str, shape, x: torch.Tensor, dtypes):
    if p is None:
        return
    if p.device != x.device:
        raise RuntimeError(f"{name} on {p.device}, input on {x.device}")
    if tuple(p.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(p.shape)}")
    if p.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {p.dtype}")


def _rows(t: torch.Tensor):
    """(tensor, row stride): `t` as rows of contiguous elements, copied only where its strides do not allow that."""
    width = t.shape[-1]
    if t.dim() == 2 and (t.stride(1) == 1 or width == 1) and (t.stride(0) >= width or t.shape[0] <= 1):
        return t, max(t.stride(0), width)
    if t.is_contiguous():
        return t, width
    return t.contiguous(), width


# ---- layer norm ------------------------------------------------------------------------------------------------------

def _layer_norm_forward(x, ldx, rows, weight, bias, eps, want_stats):
    width = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device) if want_stats else None
    affine = weight if weight is not None else bias
    code = N.DTYPE_CODES[x.dtype]
    N.launch(x.device, N.lib().dmn_layer_norm_forward, x.data_ptr(), ldx, N.ptr(weight), N.ptr(bias), y.data_ptr(), N.ptr(stats),
             rows, width, code, code if affine is None else N.DTYPE_CODES[affine.dtype], eps)
    return y, stats


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x, ldx = _rows(x)
        rows = x.numel() // x.shape[-1]
        y, stats = _layer_norm_forward(x, ldx, rows, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.ldx = ldx
        ctx.affine_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        dy, lddy = _rows(dy)
        width = x.shape[-1]
        rows = stats.shape[0]
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty(width, dtype=ctx.affine_dtype, device=x.device) if need_w else None
        db = torch.empty(width, dtype=ctx.affine_dtype, device=x.device) if need_b else None
        code, lib, ws, nbytes = N.DTYPE_CODES[x.dtype], N.lib(), None, 0
        if need_w or need_b:
            nbytes = lib.dmn_layer_norm_workspace_bytes(rows, width, code)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        N.launch(x.device, lib.dmn_layer_norm_backward, dy.data_ptr(), lddy, x.data_ptr(), ctx.ldx, N.ptr(weight),
                 stats.data_ptr(), N.ptr(dx), N.ptr(dw), N.ptr(db), rows, width, code, N.DTYPE_CODES[ctx.affine_dtype],
                 N.ptr(ws), nbytes)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of `x` [..., width] (float32, bfloat16 or float16).
    `weight` and `bias` [width] (either may be None) are of x's type or float32, both alike; their gradients come in
    that type. Rows with any stride are read in place for a 2-D `x`; other layouts are copied first."""
    _check_tensor(x, "layer_norm")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm needs a last axis of at least one element")
    width = x.shape[-1]
    _check_param(weight, "weight", (width,), x, (x.dtype, torch.float32))
    _check_param(bias, "bias", (width,), x, (x.dtype, torch.float32))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNormFunction.apply(x, weight, bias, eps)
    x, ldx = _rows(x)
    return _layer_norm_forward(x, ldx, x.numel() // width, weight, bias, eps, False)[0]


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


# ---- linear layer ------------------------------------------------------------------------------------------------------

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _linear_forward(x, ldx, weight, bias, residual, ldr, code, want_z):
    out, width = weight.shape
    rows = x.numel() // width
    y = torch.empty(x.shape[:-1] + (out,), dtype=x.dtype, device=x.device)
    z = torch.empty((rows, out), dtype=x.dtype, device=x.device) if want_z else None
    lib, dt = N.lib(), N.DTYPE_CODES[x.dtype]
    nbytes = lib.dmn_linear_forward_workspace_bytes(rows, width, out, dt)
    ws = _workspace(nbytes, x.device)
    N.launch(x.device, lib.dmn_linear_forward, x.data_ptr(), ldx, weight.data_ptr(), N.ptr(bias), N.ptr(residual), ldr, y.data_ptr(),
             N.ptr(z), rows, width, out, code, dt, N.ptr(ws), nbytes)
    return y, z


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, code):
        x, ldx = _rows(x)
        ldr = 0
        if residual is not None:
            residual, ldr = _rows(residual)
        # the value in front of the activation is all the backward needs of the forward's results
        y, z = _linear_forward(x, ldx, weight, bias, residual, ldr, code, code != 0 and any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, z)
        ctx.ldx, ctx.code = ldx, code
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            rows_dy, lddy = _rows(dy)
            out, width = weight.shape
            rows = x.numel() // width
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
            dw = torch.empty((out, width), dtype=x.dtype, device=x.device) if need_w else None
            db = torch.empty(out, dtype=x.dtype, device=x.device) if need_b else None
            lib, dt = N.lib(), N.DTYPE_CODES[x.dtype]
            nbytes = lib.dmn_linear_backward_workspace_bytes(rows, width, out, ctx.code, dt)
            ws = _workspace(nbytes, x.device)
            N.launch(x.device, lib.dmn_linear_backward, rows_dy.data_ptr(), lddy, x.data_ptr(), ctx.ldx, weight.data_ptr(), N.ptr(z),
                     N.ptr(dx), N.ptr(dw), N.ptr(db), rows, width, out, ctx.code, dt, N.ptr(ws), nbytes)
        return dx, dw, db, dy if need_r else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual in one pass: `x` [..., in], `weight` [out, in], `bias` [out], `residual` [..., out],
    all of one type (float32, bfloat16 or float16); `activation` None, 'relu', 'silu' or 'gelu' (the exact one). The sum in
    front of the activation, the activation and the residual are formed in float32 and rounded once. For the backward with
    an activation the value in front of it is kept, rounded to the type; rows with any stride are read in place for 2-D
    tensors, other layouts are copied first."""
    _check_tensor(x, "linear")
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"weight must be [out, in], got {tuple(weight.shape)}")
    out, width = weight.shape
    if x.dim() == 0 or x.shape[-1] != width:
        raise ValueError(f"expected a last axis of {width}, got {tuple(x.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    _check_param(weight, "weight", (out, width), x, (x.dtype,))
    _check_param(bias, "bias", (out,), x, (x.dtype,))
    _check_param(residual, "residual", x.shape[:-1] + (out,), x, (x.dtype,))
    weight = weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    code = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _LinearFunction.apply(x, weight, bias, residual, code)
    x, ldx = _rows(x)
    ldr = 0
    if residual is not None:
        residual, ldr = _rows(residual)
    return _linear_forward(x, ldx, weight, bias, residual, ldr, code, False)[0]


class Linear(nn.Linear):
    """torch.nn.Linear (its parameters, initialisation and state_dict) with an activation and a residual in its epilogue:
    `Linear(in, out, activation='gelu')(x)`, `Linear(in, out)(x, residual=x0)`."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: Optional[str] = None, device=None,
                 dtype=None):
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        self.activation = activation

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return linear(x, self.weight, self.bias, self.activation, residual)
