"""The optimiser with coefficients that its segments of three steps cannot hold: what orthogonalize takes, it takes.  Tolerance: test_ortho_gpu.py's
(segments of two steps, so its factor of 8 and the floor of three-step segments hold all the more)."""
import math

import pytest
import torch
from test_ortho_gpu import dev, iterate, segments_floor  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("abc", [(4.0848, -6.8946, 2.9270), (3.9, -6.0, 2.6)])
@pytest.mark.parametrize("steps", [1, 3, 5, 6])
def test_steps(dev, abc, steps):  # noqa: F811
    from taming_event_flow_amd import optim, parallel

    shapes = [(40, 70), (130, 33), (3, 20), (5,)]
    gen = torch.Generator().manual_seed(steps)
    start = [torch.randn(s, generator=gen) * 0.1 for s in shapes]
    params = [torch.nn.Parameter(p.clone().to(dev)) for p in start]
    bucket = parallel.FlatGradBucket(params)
    make = lambda: optim.FusedMuon(bucket, 0.02, nesterov=False, momentum=0.0, coefficients=abc, steps=steps)  # noqa: E731
    if abc[0] == 3.9 and steps >= 5:      # a singular value of 0.127 reaches 8.9 in the fifth step
        with pytest.raises(ValueError, match="coefficients"):
            make()
        return
    opt = make()
    grads = [torch.randn(s, generator=gen) * 0.01 for s in shapes]
    for p, g in zip(params, grads):
        p.grad.copy_(g)
    opt.step()
    assert opt.step_count.item() == 1
    for p, q, g in zip(params[:3], start, grads):
        o = iterate(g, steps, abc, 1e-7, torch.float64)
        plain = (iterate(g, steps, abc, 1e-7, torch.float32) - o).abs().max().item()
        scale = 0.02 * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        want = q.double() - scale * o
        bound = scale * (8 * plain + (segments_floor(steps, abc) + 2e-6) * o.abs().max().item()) + 2.0 ** -23 * want.abs().max().item()
        assert (p.detach().double().cpu() - want).abs().max().item() <= bound, tuple(p.shape)
