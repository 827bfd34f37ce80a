"""The optimiser step on matrices of up to 8 rows (prediction heads [2, n], narrow layers), beside larger ones.

Tolerance.  u is formed in fp32: three roundings where the 64-bit look-ahead has none, and the iteration multiplies what is rounded along small
singular values; the plain fp32 iteration on the once rounded u shows by how much, so its distance from 64 bits times 3, plus a few
roundings of the largest element, times lr * scale; and half a step of the parameter before and after the update."""
import math

import pytest
import torch
from test_ortho_gpu import ABC, dev, iterate  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = [(2, 32, 1, 1), (2, 16, 1, 1), (2, 256, 1, 1), (4, 2, 3, 3), (4, 8, 3, 3), (8, 8, 3, 3), (2, 2), (3, 1500), (1500, 3), (6,), (1, 40), (40, 70)]


def rank_one_and_noise(shape, gen, size):
    rows = shape[0]
    cols = math.prod(shape[1:])
    g = torch.randn(rows, 1, generator=gen, dtype=torch.float64) @ torch.randn(1, cols, generator=gen, dtype=torch.float64)
    return ((g + 0.01 * torch.randn(rows, cols, generator=gen, dtype=torch.float64)) * size).float().view(shape)


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("steps", [5, 12])
def test_small_matrices_are_as_near_as_plain(dev, nesterov, steps):  # noqa: F811
    from taming_event_flow_amd import optim, parallel

    lr, mu, wd = 0.02, 0.95, 0.1
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        start = [torch.randn(s, generator=gen) * 0.1 for s in SHAPES]
        params = [torch.nn.Parameter(p.clone().to(dev)) for p in start]
        bucket = parallel.FlatGradBucket(params)
        opt = optim.FusedMuon(bucket, lr, momentum=mu, nesterov=nesterov, weight_decay=wd, adam_lr=1e-3, steps=steps)
        m64 = [torch.zeros(s, dtype=torch.float64) for s in SHAPES]
        for t in range(2):
            before = [p.detach().double().cpu().clone() for p in params]
            grads = [rank_one_and_noise(s, gen, 0.01) if len(s) > 1 else torch.randn(s, generator=gen) * 0.01 for s in SHAPES]
            for p, g in zip(params, grads):
                p.grad.copy_(g)
            opt.step()
            assert not bucket.flat.any()
            for p, q, m, g in zip(params, before, m64, grads):
                m.add_((1 - mu) * (g.double() - m)) if p.dim() > 1 else None
                if p.dim() < 2 or min(p.shape[0], p.numel() // p.shape[0]) > 8:
                    continue
                u = (g.double() + mu * (m - g.double()) if nesterov else m).reshape(p.shape[0], -1)
                o = iterate(u, steps, ABC, 1e-7, torch.float64)
                plain = (iterate(u.float(), steps, ABC, 1e-7, torch.float32) - o).abs().max().item()
                scale = math.sqrt(max(1.0, p.shape[0] / (p.numel() / p.shape[0])))
                want = q * (1 - lr * wd) - lr * scale * o.view(p.shape)
                bound = lr * scale * (3 * plain + 8 * U * o.abs().max().item()) + 2 * U * (want.abs() + q.abs())
                err = (p.detach().double().cpu() - want).abs()
                assert (err <= bound).all(), (tuple(p.shape), t, (err / bound).max().item())


def test_one_form_alone(dev):  # noqa: F811
    """Only tiny, only thin, only tiled matrices; the same parameters' bits whatever stands beside them."""
    from taming_event_flow_amd import optim, parallel

    def run(shapes):
        params = [torch.nn.Parameter(torch.cos(torch.arange(math.prod(s), device=dev, dtype=torch.float32)).view(s)) for s in shapes]
        bucket = parallel.FlatGradBucket(params)
        opt = optim.FusedMuon(bucket, 0.02)
        for p in params:
            p.grad.copy_(torch.sin(torch.arange(p.numel(), device=dev) * 1.7).view(p.shape))
        opt.step()
        return [p.detach().clone() for p in params]

    together = run([(2, 40), (3, 2000), (50, 60)])
    for i, s in enumerate([(2, 40), (3, 2000), (50, 60)]):
        assert torch.equal(run([s])[0], together[i])
