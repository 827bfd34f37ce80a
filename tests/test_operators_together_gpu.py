"""Calls that the documentation allows and the other tests do not make: the same tensor twice, two streams at once, every form in one captured step,
inference mode."""
import pytest
import torch
from test_norm_gpu import check as check_norm, reference
from test_ortho_gpu import dev, matrix  # noqa: F401

pytestmark = pytest.mark.gpu


def test_one_tensor_as_input_and_residual(dev):  # noqa: F811
    from taming_event_flow_amd.models.norm import layer_norm

    gen = torch.Generator(device=dev).manual_seed(0)
    for shape in ((30, 40), (2, 24, 5, 6), (2, 24, 4, 8)):
        x = torch.randn(shape, generator=gen, device=dev, requires_grad=True)
        dy = torch.randn(shape, generator=gen, device=dev)
        y = layer_norm(x, activation="tanh", residual=x)
        want, _, _ = reference(x, None, None, x, 1, 1e-5, "tanh", dy)
        check_norm("y", y, want["y"])
        got = torch.autograd.grad(y, x, dy)[0]
        value, bound = want["dx"][0] + want["dres"][0], want["dx"][1] + want["dres"][1]
        check_norm("dx + dres", got, (value, bound + 2.0 ** -24 * value.abs()))


def test_inference_mode(dev):  # noqa: F811
    from taming_event_flow_amd.models.norm import LayerNorm
    from taming_event_flow_amd.optim import orthogonalize

    m = LayerNorm(24).to(dev)
    x = torch.randn(2, 24, 5, 6, device=dev)
    u = torch.randn(30, 50, device=dev)
    with torch.inference_mode():
        y, o = m(x, activation="relu"), orthogonalize(u)
    assert torch.equal(y, m(x, activation="relu").detach()) and torch.equal(o, orthogonalize(u))


def test_two_streams_at_once(dev):  # noqa: F811
    """Each call has a workspace of its own: lists of every form on two streams, ten times each, without a wait in between."""
    from taming_event_flow_amd.optim import orthogonalize

    lists = [[matrix("rank", *s, seed=10 * k + i).float().to(dev) for i, s in enumerate([(4, 30), (5, 4000), (40, 90), (300, 700), (200, 100)])] for k in range(2)]
    alone = [orthogonalize(us) for us in lists]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for st, us, out in zip(streams, lists, got):
            with torch.cuda.stream(st):
                out.append(orthogonalize(us))
    torch.cuda.synchronize()
    for out, want in zip(got, alone):
        assert all(torch.equal(a, b) for ys in out for a, b in zip(ys, want))


@pytest.mark.parametrize("steps", [5, 12])
def test_captured_step_of_every_form(dev, steps):  # noqa: F811
    from taming_event_flow_amd import optim, parallel

    shapes = [(2, 30), (4, 3000), (3000, 4), (40, 70), (600, 700), (9,), (1, 17), (130, 5, 3, 3)]

    def build():
        gen = torch.Generator().manual_seed(1)
        params = [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.1).to(dev)) for s in shapes]
        bucket = parallel.FlatGradBucket(params)
        return bucket, optim.FusedMuon(bucket, 0.02, adam_lr=1e-3, steps=steps, weight_decay=0.01)

    (bucket, opt), (ebucket, eager) = build(), build()
    grad = torch.sin(torch.arange(bucket.flat.numel(), device=dev) * 0.73) * 0.01
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        bucket.flat.copy_(grad)
        opt.step(1.0)
    torch.cuda.synchronize()
    ebucket.flat.copy_(grad)
    eager.step(1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(1.0)
    for k in range(3):
        bucket.flat.copy_(grad * (k + 2))
        graph.replay()
        torch.cuda.synchronize()
        ebucket.flat.copy_(grad * (k + 2))
        eager.step(1.0)
        assert torch.equal(opt.flat_p, eager.flat_p) and torch.equal(opt.m, eager.m) and torch.equal(opt.v, eager.v) and not bucket.flat.any(), k
