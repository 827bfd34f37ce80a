"""Orthogonalised updates: `orthogonalize` (Newton-Schulz) and `FusedMuon`, the optimiser step built on it.

New functionality next to parallel.FusedAdam (the reference trains with torch.optim.Adam only, train_flow.py:70): every matrix of
the network — a convolution's weight as [out, in * k * k] — is updated along the nearest semi-orthogonal matrix of its momentum, so that
all directions of a weight move at the same rate whatever the gradient's spectrum; vectors (biases, normalisation weights)
keep Adam.  The arithmetic is csrc/tef_ortho.hip.
"""

import ctypes
import math

import torch

try:
    from . import _lib
    from .parallel import FusedAdam
except ImportError:      # drop-in mode: this package's directory itself is on sys.path
    import _lib
    from parallel import FusedAdam

COEFFICIENTS = (3.4445, -4.7750, 2.0315)      # quintic with a steep slope at 0: singular values end in about [0.7, 1.2]
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # TEF_F32 / TEF_F16 / TEF_BF16 (include/tef.h)


def _aligned(nbytes, device):
    """A workspace whose first byte is 256-byte aligned -> (tensor that owns it, address)."""
    ws = torch.empty((nbytes + 255,), dtype=torch.uint8, device=device)
    return ws, (ws.data_ptr() + 255) & ~255


def _polynomial(steps, coefficients, eps):
    if int(steps) != steps or not 1 <= steps <= 32:
        raise ValueError(f"steps = {steps}: 1 to 32")
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f"coefficients = {coefficients!r}: three finite numbers")
    if not 1e-200 <= eps < 1e30:
        raise ValueError(f"eps = {eps}: positive (at least 1e-200)")
    return (int(steps),) + tuple(float(c) for c in coefficients) + (float(eps),)


def _as_batch(t):
    """[..., rows, cols] as (tensor, batch, batch stride, row stride): rows contiguous, the batch one stride apart."""
    if t.stride(-1) != 1 and t.shape[-1] > 1 or t.stride(-2) < t.shape[-1] and t.shape[-2] > 1:
        t = t.contiguous()
    rows, cols = t.shape[-2:]
    if t.dim() == 2:
        return t, 1, 0, max(t.stride(0), cols)
    if t.dim() > 3:
        try:
            t = t.view(-1, rows, cols)
        except RuntimeError:
            t = t.contiguous().view(-1, rows, cols)
    return t, t.shape[0], t.stride(0), max(t.stride(1), cols)


def orthogonalize(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """Newton-Schulz orthogonalisation: X = U / max(|U|, eps), then `steps` times X <- a X + (b A + c A A) X with A = X X^T (for a tall
    matrix X^T X), coefficients (a, b, c).  update: a matrix [rows, cols], a batch of them [..., rows, cols], or a list / tuple of such tensors
    (any mix of shapes, one type, one device: matrices of one kind in the same launches); float32, float16 or bfloat16.  -> new tensor(s)
    of the same shape and type.  The arithmetic is fp32-grade whatever the type.  A matrix of up to 64 x 320 has the same bits alone and in any
    list; of larger ones the order of sums depends on the larger ones beside it.  A zero matrix gives zeros, a NaN or an
    infinity makes its own matrix NaN.  Not differentiable."""
    many = isinstance(update, (list, tuple))
    tensors = list(update) if many else [update]
    steps, a, b, c, eps = _polynomial(steps, coefficients, eps)
    for t in tensors:
        _lib.require_device_tensor(t, "orthogonalize input")
        if t.dtype not in _DTYPES:
            raise TypeError(f"orthogonalize: float32, float16 or bfloat16 (got {t.dtype})")
        if t.dim() < 2:
            raise ValueError(f"orthogonalize: matrices [..., rows, cols], got a tensor with {t.dim()} dimension(s)")
        if t.dtype != tensors[0].dtype or t.device != tensors[0].device:
            raise ValueError("orthogonalize: the matrices of one call share a type and a device")
    out, keep, descs = [], [], []
    for t in tensors:
        o = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        out.append(o)
        if t.numel() == 0:
            continue
        s, batch, stride, ld = _as_batch(t.detach())
        keep.append(s)
        rows, cols = t.shape[-2:]
        descs.append(_lib.OrthoMatrix(s.data_ptr(), o.data_ptr(), rows, cols, ld, cols, batch, stride, rows * cols))
    if descs:
        lib = _lib.lib()
        arr = (_lib.OrthoMatrix * len(descs))(*descs)
        nbytes = lib.tef_orthogonalize_workspace_bytes(arr, len(descs))
        if nbytes == 0:
            _lib.check(-1, "tef_orthogonalize_workspace_bytes")
        first = tensors[0]
        with torch.cuda.device_of(first):
            ws, at = _aligned(nbytes, first.device)
            _lib.check(lib.tef_orthogonalize(arr, len(descs), _DTYPES[first.dtype], steps, a, b, c, eps, at, nbytes, _lib.stream_ptr()),
                       "tef_orthogonalize")
    return (out if isinstance(update, list) else tuple(out)) if many else out[0]      # (a named tuple's class takes no list)


class FusedMuon(FusedAdam):
    """Momentum with orthogonalised updates for the matrices of a FlatGradBucket, Adam for its vectors, clip_grad_norm_ and zero_grad
    in the same step, on the flat buffers (see FusedAdam: parameters become views of `flat_p`, hyper-parameters live in device
    memory, the step can be captured in a hipGraph, the caller invalidates packed weights after a step).

        m <- m + (1 - momentum) (g - m),  u = g + momentum (m - g)  (nesterov=False: u = m)
        W <- W (1 - lr weight_decay) - lr scale orthogonalize(u)

    A parameter with two dimensions or more is the matrix [shape[0], rest]; `scale` is sqrt(max(1, rows / cols)) for
    adjust_lr="original" and 0.2 sqrt(max(rows, cols)) for "match_rms_adamw" (the size of an AdamW update: learning rates carry over).  `vectors`:
    parameters that get Adam although they have two dimensions or more.  adam_lr (None: lr), betas and adam_eps are Adam's; weight_decay
    applies to the matrices only."""

    _MAX_NORM_AT = 3

    def __init__(self, bucket, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7,
                 adjust_lr="original", adam_lr=None, betas=(0.9, 0.999), adam_eps=1e-8, vectors=()):
        if adjust_lr not in ("original", "match_rms_adamw"):
            raise ValueError(f"adjust_lr = {adjust_lr!r}: 'original' or 'match_rms_adamw'")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"momentum = {momentum}: in [0, 1)")
        if not (math.isfinite(lr) and lr >= 0.0 and math.isfinite(weight_decay) and weight_decay >= 0.0):
            raise ValueError(f"lr = {lr}, weight_decay = {weight_decay}: finite, not negative")
        as_vector = {id(p) for p in vectors}
        if as_vector - {id(p) for p in bucket.params}:
            raise ValueError("vectors: parameters of the bucket (an entry is not one of them)")
        if bucket.flat.dtype != torch.float32:
            raise TypeError(f"FusedMuon: float32 parameters (got {bucket.flat.dtype})")
        self._poly = _polynomial(steps, coefficients, eps)
        if _lib.lib().tef_orthogonalize_check(*self._poly):      # (here, not in the first step, which would have been counted by then)
            raise ValueError(_lib.lib().tef_last_error().decode())
        _lib.require_device_tensor(bucket.flat, "FusedMuon gradient bucket")
        self.nesterov = bool(nesterov)
        super().__init__(bucket, lr, betas=betas, eps=adam_eps)
        self.param_groups[0].update(momentum=float(momentum), weight_decay=float(weight_decay), adam_lr=None if adam_lr is None else float(adam_lr))
        matrices, ranges, at, nvec = [], [], 0, 0
        for p in bucket.params:
            n = p.numel()
            if n and p.dim() >= 2 and id(p) not in as_vector:
                rows, cols = p.shape[0], n // p.shape[0]
                scale = math.sqrt(max(1.0, rows / cols)) if adjust_lr == "original" else 0.2 * math.sqrt(max(rows, cols))
                matrices.append(self._lib.MuonMatrix(at, rows, cols, scale))
            elif n:
                ranges.append(self._lib.MuonVector(at, n))
                nvec += n
            at += n
        self._matrices = (self._lib.MuonMatrix * len(matrices))(*matrices)
        self._vectors = (self._lib.MuonVector * len(ranges))(*ranges)
        self.v = torch.zeros((nvec,), dtype=torch.float32, device=bucket.flat.device)      # second moments of the vectors, packed
        self.hp = torch.zeros((8,), dtype=torch.float64, device=bucket.flat.device)
        nbytes = self._lib.lib().tef_muon_workspace_bytes(self._matrices, len(matrices))
        if nbytes == 0:
            self._lib.check(-1, "tef_muon_workspace_bytes")
        self._ws, self._ws_at = _aligned(nbytes, bucket.flat.device)
        self._ws_bytes = nbytes

    def _hyperparams(self, max_norm):
        g = self.param_groups[0]
        return (float(g["lr"]), float(g["momentum"]), float(g["weight_decay"]), float(max_norm),
                float(g["lr"] if g["adam_lr"] is None else g["adam_lr"]), float(g["betas"][0]), float(g["betas"][1]), float(g["eps"]))

    def state_dict(self):
        """The momentum of the matrices and first moments of the vectors (flat, in parameter order), the vectors' second moments (packed),
        the step count, and the hyper-parameters."""
        return {"state": {"momentum": self.m.detach().clone(), "exp_avg_sq": self.v.detach().clone(), "step": self.step_count.detach().clone()},
                "param_groups": [{k: v for k, v in self.param_groups[0].items() if k != "params"}]}

    def load_state_dict(self, sd):
        st = sd["state"]
        if "momentum" not in st or st["momentum"].numel() != self.m.numel() or st["exp_avg_sq"].numel() != self.v.numel():
            raise ValueError("FusedMuon.load_state_dict: state of another optimiser or parameter set")
        self.m.copy_(st["momentum"].reshape(-1))
        self.v.copy_(st["exp_avg_sq"].reshape(-1))
        self.step_count.copy_(st["step"].reshape(-1))
        for k, v in sd["param_groups"][0].items():
            if k != "params":
                self.param_groups[0][k] = tuple(v) if k == "betas" else v

    def step(self, max_norm=None):
        """One step on the (already reduced) flat gradient, see FusedAdam.step: clip to `max_norm`, update, clear -> the norm before clipping."""
        with torch.cuda.device_of(self.flat_p):
            return super().step(max_norm)

    def _update(self, stream):
        code = self._lib.lib().tef_muon_step(self.flat_p.data_ptr(), self.bucket.flat.data_ptr(), self.m.data_ptr(), self.v.data_ptr(),
                                             self._matrices, len(self._matrices), self._vectors, len(self._vectors),
                                             self.norm.data_ptr(), self.hp.data_ptr(), self.step_count.data_ptr(), int(self.nesterov),
                                             *self._poly, self._ws_at, self._ws_bytes, stream)
        self._lib.check(code, "tef_muon_step")
