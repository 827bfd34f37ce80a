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


def test_heads_left_to_adam_by_name(dev):  # noqa: F811
    """A Trainer's config: `vectors: [arch.preds]` gives the prediction heads Adam (a first step of at most adam_lr), the rest orthogonalised ones."""
    import copy

    from taming_event_flow_amd import train

    cfg = copy.deepcopy(train.DEFAULT_CONFIG)
    cfg["data"]["passes_loss"] = 2
    cfg["loader"].update(batch_size=1, resolution=[32, 32], max_num_grad_events=200)
    cfg["model"].update(base_channels=8)
    cfg["optimizer"] = dict(name="Muon", lr=0.5, adam_lr=1e-4, vectors=["arch.preds"])
    torch.manual_seed(0)
    tr = train.Trainer(cfg, dev)
    src = train.SyntheticSequences(cfg, dev, 300, seq_len=10 ** 9)
    before = {n: p.detach().clone() for n, p in tr.model.named_parameters()}
    tr.step(src.next(), new_seq=True), tr.step(src.next())
    moved = {n: (p.detach() - before[n]).abs().max().item() for n, p in tr.model.named_parameters()}
    heads = [n for n in moved if ".preds." in n]
    assert len(heads) == 8 and all(moved[n] <= 1.01e-4 for n in heads) and max(moved[n] for n in heads) > 0
    assert any(v > 1e-2 for n, v in moved.items() if n not in heads)
    tr.close()
