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


def _check_param(p: torch.Tensor, name: str, shape, x: torch.Tensor, other=None):
    """`p` on x's device, of `shape` and of x's type (or `other`)."""
    if p.device != x.device:
        raise RuntimeError(f"{name} on {p.device}, input on {x.device}")
    if p.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(p.shape)}")
    if p.dtype != x.dtype and p.dtype != other:
        raise ValueError(f"{name} must be {x.dtype}{'' if other is None else f' or {other}'}, got {p.dtype}")


def _rows(t: torch.Tensor):
    """(tensor, row stride): `t` as rows of contiguous elements, copied only where its strides do not allow that."""
    width = t.shape[-1]
    if t.is_contiguous():
        return t, width
    if t.dim() == 2 and (t.stride(1) == 1 or width == 1) and t.stride(0) >= width:
        return t, t.stride(0)
    return t.contiguous(), width


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


# ---- layer norm ------------------------------------------------------------------------------------------------------

def _layer_norm_forward(x, ldx, weight, bias, eps, want_stats):
    width = x.shape[-1]
    rows = x.numel() // width
    y = _empty_like(x)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device) if want_stats else None
    code = N.DTYPE_CODES[x.dtype]
    affine = code if weight is bias is None else N.DTYPE_CODES[(bias if weight is None else weight).dtype]
    N.launch(x.get_device(), N.lib().dmn_layer_norm_forward, x.data_ptr(), ldx, None if weight is None else weight.data_ptr(),
             None if bias is None else bias.data_ptr(), y.data_ptr(), None if stats is None else stats.data_ptr(), rows, width, code,
             affine, eps)
    return y, stats, rows, code, affine


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x, ldx = _rows(x)
        y, stats, rows, code, affine = _layer_norm_forward(x, ldx, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.plan = ldx, rows, code, affine
        return y

    @staticmethod
    def backward(ctx, dy):
        # the decorator that refuses a second differentiation costs more than the work below where nobody asks for one
        return _LayerNormFunction._once(ctx, dy) if torch.is_grad_enabled() else _LayerNormFunction._gradients(ctx, dy)

    @staticmethod
    def _gradients(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        ldx, rows, code, affine = ctx.plan
        dy, lddy = _rows(dy)
        width = x.shape[-1]
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx = _empty_like(x) if need_x else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(bias) if need_b else None
        lib, ws, nbytes = N.lib(), None, 0
        if need_w or need_b:
            nbytes = lib.dmn_layer_norm_workspace_bytes(rows, width, code)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        N.launch(x.get_device(), lib.dmn_layer_norm_backward, dy.data_ptr(), lddy, x.data_ptr(), ldx,
                 None if weight is None else weight.data_ptr(), stats.data_ptr(), None if dx is None else dx.data_ptr(),
                 None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(), rows, width, code, affine,
                 None if ws is None else ws.data_ptr(), nbytes)
        return dx, dw, db, None

    _once = staticmethod(once_differentiable(_gradients.__func__))


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of `x` [..., width] (float32, bfloat16 or float16).
    `weight` and `bias` [width] (either may be None) are of x's type or float32, both alike; their gradients come in
    that type. Rows with any stride are read in place for a 2-D `x`; other layouts are copied first."""
    _check_tensor(x, "layer_norm")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm needs a last axis of at least one element")
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    shape, grad = x.shape[-1:], x.requires_grad
    if weight is not None:
        _check_param(weight, "weight", shape, x, torch.float32)
        weight, grad = weight.contiguous(), grad or weight.requires_grad
    if bias is not None:
        _check_param(bias, "bias", shape, x, torch.float32)
        if weight is not None and weight.dtype != bias.dtype:
            raise ValueError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
        bias, grad = bias.contiguous(), grad or bias.requires_grad
    if grad and torch.is_grad_enabled():
        return _LayerNormFunction.apply(x, weight, bias, eps)
    x, ldx = _rows(x)
    return _layer_norm_forward(x, ldx, weight, bias, eps, False)[0]


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


def _linear_forward(x, ldx, weight, bias, residual, ldr, activation, want_z):
    out, width = weight.shape
    rows = x.numel() // width
    y = torch.empty(x.shape[:-1] + (out,), dtype=x.dtype, device=x.device)
    z = torch.empty_like(y) if want_z else None
    lib, code = N.lib(), N.DTYPE_CODES[x.dtype]
    px, pw = x.data_ptr(), weight.data_ptr()
    nbytes = lib.dmn_linear_forward_workspace_bytes(px, ldx, pw, rows, width, out, code)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    N.launch(x.get_device(), lib.dmn_linear_forward, px, ldx, pw, None if bias is None else bias.data_ptr(),
             None if residual is None else residual.data_ptr(), ldr, y.data_ptr(), None if z is None else z.data_ptr(), rows, width,
             out, activation, code, None if ws is None else ws.data_ptr(), nbytes)
    return y, z, rows, code


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        x, ldx = _rows(x)
        ldr = 0
        if residual is not None:
            residual, ldr = _rows(residual)
        # the value in front of the activation is all the backward needs of the forward's results
        y, z, rows, code = _linear_forward(x, ldx, weight, bias, residual, ldr, activation,
                                           activation != 0 and any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, bias, z)
        ctx.plan = ldx, rows, code, activation
        return y

    @staticmethod
    def backward(ctx, dy):
        return _LinearFunction._once(ctx, dy) if torch.is_grad_enabled() else _LinearFunction._gradients(ctx, dy)

    @staticmethod
    def _gradients(ctx, dy):
        x, weight, bias, z = ctx.saved_tensors
        ldx, rows, code, activation = ctx.plan
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dx = dw = db = None
        if need_x or need_w or need_b:
            rows_dy, lddy = _rows(dy)
            out, width = weight.shape
            dx = _empty_like(x) if need_x else None
            dw = torch.empty_like(weight) if need_w else None
            db = torch.empty_like(bias) if need_b else None
            lib = N.lib()
            pd, px, pw = rows_dy.data_ptr(), x.data_ptr(), weight.data_ptr()
            nbytes = lib.dmn_linear_backward_workspace_bytes(pd, lddy, px, ldx, pw, rows, width, out, activation, code)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
            N.launch(x.get_device(), lib.dmn_linear_backward, pd, lddy, px, ldx, pw,
                     None if z is None else z.data_ptr(), None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
                     None if db is None else db.data_ptr(), rows, width, out, activation, code, None if ws is None else ws.data_ptr(),
                     nbytes)
        return dx, dw, db, dy if need_r else None, None

    _once = staticmethod(once_differentiable(_gradients.__func__))


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
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    _check_param(weight, "weight", weight.shape, x)
    weight, grad = weight.contiguous(), x.requires_grad or weight.requires_grad
    if bias is not None:
        _check_param(bias, "bias", (out,), x)
        bias, grad = bias.contiguous(), grad or bias.requires_grad
    if residual is not None:
        _check_param(residual, "residual", x.shape[:-1] + (out,), x)
        grad = grad or residual.requires_grad
    if grad and torch.is_grad_enabled():
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
