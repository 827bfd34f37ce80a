"""Orthogonalisation and optimiser step through every tile size and cut of the products.  test_ortho_plans.py checks, without a device, that these
cases reach every kernel there is.  Tolerances: test_ortho_gpu.py."""
import math

import pytest
import torch
from test_ortho_gpu import ABC, check, dev, iterate, matrix, segments_floor  # noqa: F401

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# lists of (batch, rows, cols), type
CASES = {
    "large": ([(1, 2048, 2048)], "f32"), "large_bf16": ([(1, 2048, 2048)], "bf16"), "large_f16": ([(1, 2048, 2048)], "f16"),
    "odd": ([(1, 1411, 2053)], "f32"), "odd_tall": ([(1, 2053, 1411)], "f32"), "odd_tall_bf16": ([(1, 2053, 1411)], "bf16"),
    "gates": ([(3, 256, 4608)], "f32"), "batch": ([(16, 256, 4096)], "f32"), "batch_tall": ([(16, 1300, 200)], "f32"),
    "long": ([(1, 130, 50000)], "f32"), "long_tall_f16": ([(1, 50000, 130)], "f16"),
    "edge": ([(1, 1030, 1100)], "f32"), "edge_f16": ([(1, 1030, 1100)], "f16"), "small_tiles_bf16": ([(2, 200, 333)], "bf16"),
    "list": ([(1, 512, 2304), (2, 300, 500), (1, 1000, 70), (1, 66, 3000)], "f32"), "list_large": ([(1, 2048, 2048), (1, 2000, 2100)], "f32"),
    "many": ([(40, 300, 310)], "f32"),
}
MUON = {
    "gates_and_blocks": [(512, 4608)] * 9 + [(512, 9216), (64, 18), (2, 256)], "one_large": [(2048, 2048)], "one_odd_tall": [(1500, 1411)],
    "narrow": [(16, 45), (32, 144), (64, 288), (128, 576), (2, 16)], "one": [(130, 70)],
}


@pytest.mark.parametrize("name", CASES)
def test_tiles(dev, name):  # noqa: F811
    from taming_event_flow_amd.optim import orthogonalize

    shapes, dtype = CASES[name]
    us = []
    for i, (b, r, c) in enumerate(shapes):
        u = torch.stack([matrix("rank", r, c, seed=i + 10 * k) for k in range(min(b, 3))]).to(DTYPES[dtype])
        us.append(u.repeat((b + 2) // 3, 1, 1)[:b].to(dev) if b > 1 else u[0].to(dev))
    got = orthogonalize(us) if len(us) > 1 else [orthogonalize(us[0])]
    for u, y in zip(us, got):
        if u.dim() == 2:
            check(y, u)
            continue
        for k in range(min(3, len(u))):
            check(y[k], u[k])
            check(y[len(u) - 3 + k], u[len(u) - 3 + k]) if len(u) > 3 else None
    again = orthogonalize(us) if len(us) > 1 else [orthogonalize(us[0])]
    assert all(torch.equal(y, z) for y, z in zip(got, again))


@pytest.mark.parametrize("name", MUON)
def test_optimiser(dev, name):  # noqa: F811
    from taming_event_flow_amd import optim, parallel

    lr, wd = 0.02, 0.1
    gen = torch.Generator().manual_seed(7)
    start = [torch.randn(s, generator=gen) * 0.1 for s in MUON[name]]
    params = [torch.nn.Parameter(p.clone().to(dev)) for p in start]
    bucket = parallel.FlatGradBucket(params)
    opt = optim.FusedMuon(bucket, lr, weight_decay=wd)
    grads = [(matrix("rank", *s, seed=i) * 0.01).float() for i, s in enumerate(MUON[name])]
    for p, g in zip(params, grads):
        p.grad.copy_(g)
    opt.step()
    assert not bucket.flat.any()
    for p, q, g in zip(params, start, grads):
        u = (0.05 * 0.95 + 0.05) * g.double()
        o = iterate(u, 5, ABC, 1e-7, torch.float64)
        plain = (iterate(u.float(), 5, ABC, 1e-7, torch.float32) - o).abs().max().item()
        scale = lr * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        want = q.double() * (1 - lr * wd) - scale * o
        bound = scale * (8 * plain + (segments_floor(5, ABC) + 2e-6) * o.abs().max().item()) + 2.0 ** -23 * want.abs().max().item()
        assert (p.detach().double().cpu() - want).abs().max().item() <= bound, tuple(p.shape)
