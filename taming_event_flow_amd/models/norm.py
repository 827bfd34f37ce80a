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


_TORCH = {code: dtype for dtype, code in _DTYPES.items()}


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, dim, eps, act, keep):
        # a map in channels-last memory is a matrix of rows as it stands; anything else is taken in x's own dimension order
        shape = x.shape
        if dim == len(shape) - 1:
            xc, rows = x.contiguous(), True
            like = xc
        elif x.is_contiguous():
            xc, rows = x, False
            like = x
        else:
            last = x.movedim(dim, -1)
            rows = last.is_contiguous()
            xc = last if rows else x.contiguous()
            like = x if rows else xc
        rc = residual
        if rc is not None:
            rc = (rc.movedim(dim, -1) if rows else rc).contiguous()
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        C = shape[dim]
        inner = 1 if rows else math.prod(shape[dim + 1:])
        n = x.numel() // C      # positions
        vec = w if w is not None else b
        dtype = _DTYPES[x.dtype]
        d = _lib.NormDesc(n // inner if n else 0, inner if n else 1, C, dtype, dtype if vec is None else _DTYPES[vec.dtype], _lib.ACT[act], eps)
        # results are tensors of their own in `like`'s shape and order, no views: the caller may change them in place
        y = torch.empty_like(like)
        stats = torch.empty((2 * n,), dtype=torch.float32, device=x.device) if keep else None
        at = stats.data_ptr() if keep else None
        with torch.cuda.device_of(x):
            code = _lib.lib().tef_layer_norm_forward(ctypes.byref(d), xc.data_ptr(), _ptr(w), _ptr(b), _ptr(rc), y.data_ptr(), at,
                                                     at + 4 * n if keep else None, _lib.stream_ptr())
        _lib.check(code, "tef_layer_norm_forward")
        if keep:
            if act is None:      # (only an activation's slope needs them again)
                b = rc = None
            ctx.save_for_backward(xc, w, b, rc, stats)
            ctx.info = d, n, rows, dim, shape, like.stride()
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():      # (create_graph=True)
            raise RuntimeError("layer_norm is differentiable once: its backward pass has no gradient of its own")
        xc, w, b, rc, stats = ctx.saved_tensors
        d, n, rows, dim, shape, strides = ctx.info
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy = (dy.movedim(dim, -1) if rows else dy).contiguous()
        dx, dr = (torch.empty_strided(shape, strides, dtype=xc.dtype, device=xc.device) if need else None for need in (need_x, need_r))
        lib, dw, db, ws, nbytes = _lib.lib(), None, None, None, 0
        if need_w or need_b:
            dw = torch.empty((d.channels,), dtype=_TORCH[d.wdtype], device=xc.device) if need_w else None
            db = torch.empty((d.channels,), dtype=_TORCH[d.wdtype], device=xc.device) if need_b else None
            nbytes = lib.tef_layer_norm_workspace_bytes(ctypes.byref(d))
            ws = torch.empty((nbytes,), dtype=torch.uint8, device=xc.device)
        at = stats.data_ptr()
        with torch.cuda.device_of(xc):
            code = lib.tef_layer_norm_backward(ctypes.byref(d), xc.data_ptr(), _ptr(w), _ptr(b), _ptr(rc), at, at + 4 * n, dy.data_ptr(),
                                               _ptr(dx), _ptr(dr), _ptr(dw), _ptr(db), _ptr(ws), nbytes, _lib.stream_ptr())
        _lib.check(code, "tef_layer_norm_backward")
        return dx, dw, db, dr, None, None, None, None


def layer_norm(x, weight=None, bias=None, dim=1, eps=1e-5, activation=None, residual=None):
    """act(normalise(x) * weight + bias + residual), normalised over the dimension `dim` at every position of the others
    (dim=1: the channels of feature maps [B, C, H, W]; dim=-1: rows).  x: float32, float16 or bfloat16 on a HIP device, any
    strides (a contiguous or channels-last x is read in place and the result has its memory order; of any other x it is contiguous); weight, bias: [C], of x's
    type or float32 (both the same), or None; residual: like x, or None; activation: "relu", "tanh", "sigmoid" or None.
    Statistics are fp32 whatever the type; at most 2^30 elements are
    normalised together.  Differentiable once, with respect to x, weight, bias and residual; the
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
    if C > 2 ** 30:
        raise ValueError(f"layer_norm: {C} elements to normalise over (2^30 at most)")
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
    # (a parameter asks for gradients under no_grad too: what the backward pass needs is kept only where there will be one)
    keep = torch.is_grad_enabled() and (x.requires_grad or weight is not None and weight.requires_grad or bias is not None and bias.requires_grad
                                        or residual is not None and residual.requires_grad)
    return _LayerNormFn.apply(x, weight, bias, residual, dim, float(eps), activation, keep)


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
