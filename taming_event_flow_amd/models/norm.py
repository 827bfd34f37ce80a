"""Layer normalisation of the network's features, fused with the activation and the residual sum that follow it.

The reference's layers take a ``norm`` argument ("BN" / "IN", models/submodules.py:33-62) that RecEVFlowNet leaves at None;
both kinds tie a sample's output to the batch or to the map it came with.  `LayerNorm` normalises the channels of every
position on its own — the same arithmetic for one sample, a batch, or a whole loss window decoded at once — and is what the
layers of this package build for ``norm="LN"``.  The arithmetic is csrc/tef_norm.hip.
"""

import ctypes
import math

import torch
import torch.nn as nn

try:
    from .. import _lib
except ImportError:      # drop-in mode: this package's directory itself is on sys.path
    import _lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # TEF_F32 / TEF_F16 / TEF_BF16 (include/tef.h)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _rows_last(t, dim):
    return t.movedim(dim, -1)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, dim, eps, act):
        lib = _lib.lib()
        # a map in channels-last memory is a matrix of rows as it stands; anything else is taken in x's own dimension order
        last = _rows_last(x, dim)
        rows = last.is_contiguous()
        arrange = (lambda t: _rows_last(t, dim).contiguous()) if rows else (lambda t: t.contiguous())
        shape = x.shape
        xc = arrange(x)
        rc = arrange(residual) if residual is not None else None
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        outer, inner = (math.prod(xc.shape[:-1]), 1) if rows else (math.prod(shape[:dim]), math.prod(shape[dim + 1:]))
        if inner == 0:
            outer, inner = 0, 1
        vec = w if w is not None else b
        d = _lib.NormDesc(outer, inner, shape[dim], _DTYPES[x.dtype], _DTYPES[vec.dtype if vec is not None else x.dtype], _lib.ACT[act],
                          eps)
        y = torch.empty_like(xc)
        keep = any(ctx.needs_input_grad)
        stats = torch.empty((2, outer * inner), dtype=torch.float32, device=x.device) if keep else None
        n = 4 * outer * inner
        with torch.cuda.device_of(x):
            rc_ = lib.tef_layer_norm_forward(ctypes.byref(d), xc.data_ptr(), _ptr(w), _ptr(b), _ptr(rc), y.data_ptr(),
                                             stats.data_ptr() if keep else None, stats.data_ptr() + n if keep else None,
                                             _lib.stream_ptr())
        _lib.check(rc_, "tef_layer_norm_forward")
        if keep:
            need_z = act is not None
            ctx.save_for_backward(xc, w, b if need_z else None, rc if need_z else None, stats)
            ctx.desc, ctx.rows, ctx.dim, ctx.shape, ctx.vec = d, rows, dim, shape, (weight is not None, bias is not None)
        return y.movedim(-1, dim) if rows else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        lib = _lib.lib()
        xc, w, b, rc, stats = ctx.saved_tensors
        d = ctx.desc
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dyc = (_rows_last(dy, ctx.dim) if ctx.rows else dy).contiguous()
        wdtype = {v: k for k, v in _DTYPES.items()}[d.wdtype]
        new = lambda need: torch.empty_like(xc) if need else None  # noqa: E731
        vec = lambda need: torch.empty((d.channels,), dtype=wdtype, device=xc.device) if need else None  # noqa: E731
        dx, dr, dw, db = new(need_x), new(need_r), vec(need_w), vec(need_b)
        nbytes = lib.tef_layer_norm_workspace_bytes(ctypes.byref(d)) if need_w or need_b else 0
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=xc.device) if nbytes else None
        with torch.cuda.device_of(xc):
            rc_ = lib.tef_layer_norm_backward(ctypes.byref(d), xc.data_ptr(), _ptr(w), _ptr(b), _ptr(rc), stats.data_ptr(),
                                              stats.data_ptr() + 4 * d.outer * d.inner, dyc.data_ptr(), _ptr(dx), _ptr(dr),
                                              _ptr(dw), _ptr(db), _ptr(ws), nbytes, _lib.stream_ptr())
        _lib.check(rc_, "tef_layer_norm_backward")
        back = (lambda t: t.movedim(-1, ctx.dim) if t is not None and ctx.rows else t)
        return back(dx), dw, db, back(dr), None, None, None


def layer_norm(x, weight=None, bias=None, dim=1, eps=1e-5, activation=None, residual=None):
    """act(normalise(x) * weight + bias + residual), normalised over the dimension `dim` at every position of the others
    (dim=1: the channels of feature maps [B, C, H, W]; dim=-1: rows).  x: float32, float16 or bfloat16 on a HIP device, any
    strides (a contiguous or channels-last x is read in place; the result has x's memory order); weight, bias: [C], of x's
    type or float32 (both the same), or None; residual: like x, or None; activation: "relu", "tanh", "sigmoid" or None.
    Statistics are fp32 whatever the type.  Differentiable once, with respect to x, weight, bias and residual; the
    gradients of weight and bias are reproducible bit for bit."""
    _lib.require_device_tensor(x, "layer_norm input")
    if x.dtype not in _DTYPES:
        raise TypeError(f"layer_norm: float32, float16 or bfloat16 (got {x.dtype})")
    if not -x.dim() <= dim < x.dim():
        raise IndexError(f"layer_norm: dimension {dim} of a tensor with {x.dim()} dimensions")
    dim %= x.dim()
    C = x.shape[dim]
    if C == 0:
        raise ValueError("layer_norm: nothing to normalise over (the dimension has size 0)")
    if not (math.isfinite(eps) and 0.0 <= eps < 1e30):
        raise ValueError(f"layer_norm: eps = {eps}")
    if activation not in _lib.ACT:
        raise NotImplementedError(f"layer_norm: activation {activation!r} (relu / tanh / sigmoid / None)")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (C,):
            raise ValueError(f"layer_norm: {name} of shape {tuple(t.shape)} for {C} channels")
        if t.device != x.device:
            raise RuntimeError(f"layer_norm: {name} on {t.device}, input on {x.device}")
        if t.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"layer_norm: {name} of type {t.dtype} for an input of type {x.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"layer_norm: weight of type {weight.dtype}, bias of type {bias.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"layer_norm: residual {tuple(residual.shape)} {residual.dtype} on {residual.device} for an input "
                         f"{tuple(x.shape)} {x.dtype} on {x.device}")
    return _LayerNormFn.apply(x, weight, bias, residual, dim, float(eps), activation)


class LayerNorm(nn.Module):
    """layer_norm with parameters: weight (ones) and bias (zeros) of `channels` elements."""

    def __init__(self, channels, dim=1, eps=1e-5):
        super().__init__()
        self.channels, self.dim, self.eps = int(channels), dim, eps
        self.weight = nn.Parameter(torch.ones(self.channels))
        self.bias = nn.Parameter(torch.zeros(self.channels))

    def extra_repr(self):
        return f"{self.channels}, dim={self.dim}, eps={self.eps}"

    def forward(self, x, residual=None, activation=None):
        return layer_norm(x, self.weight, self.bias, self.dim, self.eps, activation, residual)
