#!/usr/bin/env python3
"""Host-side sanitizer run of the normalisation and orthogonalisation entry points WITHOUT a GPU (as dry_run_driver.py: instrumented library,
launches that do nothing, host tensors in the place of device tensors): every kernel form's plan, workspace and argument lists.  The numbers are
garbage; any report aborts the process."""
import ctypes
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)
assert "TEF_HIP_LIB" in os.environ, "run through tests/asan/run_host_asan.sh"
from taming_event_flow_amd import _lib  # noqa: E402

_lib.require_device_tensor = lambda t, name: t
_lib.stream_ptr = lambda: None
torch.cuda.is_current_stream_capturing = lambda: False
from taming_event_flow_amd import optim, parallel  # noqa: E402
from taming_event_flow_amd.models.norm import layer_norm  # noqa: E402

stub = ctypes.CDLL(os.environ["TEF_HIP_STUB"])

for dtype in (torch.float32, torch.float16, torch.bfloat16):
    for shape in ((1, 1), (5, 2), (257, 3), (33, 64), (2, 256), (3, 257), (5, 1030), (2, 4099), (2, 8192), (3, 8193), (1, 1, 2, 2), (2, 3, 5, 7), (1, 512, 8, 8),
                  (2, 258, 3, 5), (1, 64, 1, 3), (1, 1030, 2, 2), (2, 1100, 1, 3), (1, 9000, 1, 3), (0, 8), (2, 8, 0, 4)):
        x, w, b = torch.zeros(shape, dtype=dtype, requires_grad=True), torch.ones(shape[1], requires_grad=True), torch.zeros(shape[1], requires_grad=True)
        for act in (None, "tanh"):
            y = layer_norm(x, w, b, activation=act, residual=x.detach())
            torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
print("ok: layer norm", flush=True)

SHAPES = [(1, 1), (8, 8), (3, 70), (8, 1024), (8, 1025), (2, 70001), (70001, 2), (9, 9), (64, 320), (320, 64), (64, 321), (65, 65), (200, 333), (1030, 1100),
          (1411, 2053), (2053, 1411), (256, 4608), (130, 50000), (2048, 2048)]
for steps in (1, 5, 12, 32):
    for s in SHAPES:
        optim.orthogonalize(torch.zeros(s), steps=steps)
    optim.orthogonalize([torch.zeros(s) for s in SHAPES[:14]] * 5, steps=steps)
    optim.orthogonalize([torch.zeros(3, 100, 120), torch.zeros(2, 2, 8, 2000), torch.zeros(40, 20, 30)], steps=steps)
optim.orthogonalize([torch.zeros(4 + k % 90, 6 + k % 70, dtype=torch.bfloat16) for k in range(300)])
print("ok: orthogonalize", flush=True)

for shapes in ([(64, 64, 3, 3), (64,), (2, 9, 1, 1), (5, 7), (3000, 4), (1, 1)], [(512, 4608)] * 9 + [(512,)] * 9, [(6, 10)] * 150 + [(80, 90)] * 70 + [(5,)] * 230, [(4,)], [(9, 9)]):
    params = [torch.nn.Parameter(torch.zeros(s)) for s in shapes]
    for steps, abc in ((5, optim.COEFFICIENTS), (6, (4.0848, -6.8946, 2.9270)), (1, optim.COEFFICIENTS), (32, (2.0, -1.5, 0.5))):
        opt = optim.FusedMuon(parallel.FlatGradBucket(params), 0.02, steps=steps, coefficients=abc)
        opt.step(1.0)
print("ok: FusedMuon", flush=True)

plan = _lib.OrthoPlan()
arr = (_lib.OrthoMatrix * len(SHAPES))(*[_lib.OrthoMatrix(1, 1, r, c, c, c, 1, 0, 0) for r, c in SHAPES])
for optimiser in (0, 1):
    for i in range(len(SHAPES)):
        assert _lib.lib().tef_orthogonalize_plan(arr, len(SHAPES), i, optimiser, ctypes.byref(plan)) == 0
print("HOST SANITIZER RUN CLEAN (operators)", flush=True)
