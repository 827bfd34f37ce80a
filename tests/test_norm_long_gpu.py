"""Layer normalisation of very long rows against 64 bits on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    import __graft_entry__ as g

    g.build()
    return torch.device("cuda:0")


def test_more_columns_than_a_launch_has_threads(dev):
    """2^27 + 77 channels: the sums over rows have 2^28 columns, joined by workgroups of 1024 threads for 64 columns each; and a sum of
    2^27 terms of one sign, where one running fp32 sum a thread (2^19 terms) would be off by parts in 10^5."""
    from taming_event_flow_amd.models.norm import layer_norm

    C = 2 ** 27 + 77
    gen = torch.Generator(device=dev).manual_seed(0)
    x = (torch.rand((1, C), generator=gen, device=dev) + 0.5).requires_grad_(True)
    w = torch.ones(C, device=dev, requires_grad=True)
    b = torch.zeros(C, device=dev, requires_grad=True)
    dy = torch.rand((1, C), generator=gen, device=dev) + 1
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert torch.equal(db, dy[0])      # one row: the gradient itself
    x64 = x.detach().double()
    mean, var = x64.mean(), x64.var(unbiased=False)
    rstd = 1 / (var + 1e-5).sqrt()
    u = (x64 - mean) * rstd
    # mean is off by half a step (at most 2^-24 of values below 2), x - mean by another, u |u| <= 1.8 by rstd's few roundings
    U = 2.0 ** -24
    du = 2 * 2 * U * rstd + 8 * U * 1.8
    assert ((y.detach() - u).abs().max() <= du).item()
    assert ((dw - dy[0] * u[0]).abs().max() <= 2 * du + 4 * U).item()
    d64 = dy.double()
    s1, s2 = d64.mean(), (d64 * u).mean()
    want = rstd * (d64 - s1 - u * s2)
    # g, s1 and u s2 with a few roundings each, u off by du in the last two; rstd relative
    bound = rstd * (8 * U * (d64.abs().max() + s1.abs() + 1.8 * s2.abs()) + du * (s2.abs() + d64.abs().mean())) + 8 * U * want.abs().max()
    assert ((dx - want).abs().max() <= bound).item()


CASES = [((70001, 32768), lambda t: t[-3:]), ((300007, 8192), lambda t: t[-3:]), ((33, 1024, 256, 257), lambda t: t[-1:, :, -2:]),
         ((33, 1024, 255, 257), lambda t: t[-1:, :, -2:]), ((5, 9000, 223, 223), lambda t: t[-1:, :, -1:])]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_gradients_past_32_bits(dev, case):
    """More than 2^31 elements, in the rows' and the maps' forms and the long one: every gradient at the last rows / positions, and those of the
    vectors, to which only they contribute (the rest has a gradient of zero).  Bounds: test_norm_gpu.py."""
    from test_norm_gpu import check, reference
    from taming_event_flow_amd.models.norm import layer_norm

    shape, tail = CASES[case]
    C = shape[1]
    assert torch.Size(shape).numel() > 2 ** 31
    gen = torch.Generator(device=dev).manual_seed(case)
    x, r, dy = (torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(3))
    parts = []
    for t in (x, r, dy):
        parts.append(torch.randn(tail(t).shape, generator=gen, device=dev).to(t.dtype))
        tail(t).copy_(parts[-1])
    w, b = torch.linspace(0.5, 1.5, C, device=dev), torch.linspace(-1, 1, C, device=dev)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    y = layer_norm(x, w, b, activation="tanh", residual=r)
    want, _, _ = reference(parts[0], w, b, parts[1], 1, 1e-5, "tanh", parts[2])
    check("y", tail(y.detach()), want["y"])
    grads = torch.autograd.grad(y, leaves, dy)
    del y
    for name, g in zip(("dx", "dw", "db", "dres"), grads):
        check(name, tail(g) if g.dim() > 1 else g, want[name])
    for g in (grads[0], grads[3]):
        assert not g[0].any()
