"""Layer normalisation where the mean is large against the spread: the mean's own rounding is what could show."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    import __graft_entry__ as g

    g.build()
    return torch.device("cuda:0")


SHAPES = [(5, 48), (3, 300), (7, 1030), (2, 5001), (2, 9001), (2, 48, 3, 5), (1, 258, 4, 4), (2, 600, 3, 3), (1, 9000, 2, 2)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("value", [1000.1, -77.7, 3.3e7, 1e-3])
def test_constant_rows_give_the_bias(dev, shape, value):
    """All values equal, not a number that sums exactly.  With at most D = 100 roundings on the way of a sum (long rows: sums in 64 bits)
    a mean is off by D U |x|; taken again of x - mean, by D U of that, and eps makes at most 1 / sqrt(eps) of it.  The gradient with respect to x is
    rstd (h - mean h), a few roundings and the join's D U."""
    from taming_event_flow_amd.models.norm import layer_norm

    eps, D = 1e-5, 100
    C, lane = shape[1], [1, -1] + [1] * (len(shape) - 2)
    gen = torch.Generator(device=dev).manual_seed(1)
    x = torch.full(shape, value, device=dev, requires_grad=True)
    w = 1 + 0.3 * torch.randn(C, generator=gen, device=dev)
    b = 0.2 * torch.randn(C, generator=gen, device=dev)
    dy = torch.randn(shape, generator=gen, device=dev)
    y = layer_norm(x, w, b, eps=eps)
    off = (D * U) ** 2 * abs(float(x.detach().reshape(-1)[0])) / eps ** 0.5
    b64 = b.double().view(lane)
    assert ((y.detach().double() - b64).abs() <= off * w.double().abs().view(lane) + U * b64.abs()).all()
    dx, = torch.autograd.grad(y, x, dy)
    h = dy.double() * w.double().view(lane)
    want = (h - h.mean(1, keepdim=True)) / eps ** 0.5
    bound = ((8 * U + off) * h.abs() + (D * U + off) * h.abs().mean(1, keepdim=True) * (1 + off)) / eps ** 0.5 + 8 * U * want.abs()
    assert ((dx.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("shape", SHAPES)
def test_far_offset(dev, shape):
    """A mean of 5e4 on a spread of 1: x - mean is exact to U |x| D U, what is left are the roundings of u's own size."""
    from taming_event_flow_amd.models.norm import layer_norm

    gen = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(shape, generator=gen, device=dev) + 5e4
    y = layer_norm(x).double()
    x64 = x.double()
    mean, var = x64.mean(1, keepdim=True), x64.var(1, unbiased=False, keepdim=True)
    u = (x64 - mean) / (var + 1e-5).sqrt()
    D = 100
    du = D * U * D * U * 6e4 / var.sqrt() + (2 * D + 8) * U * u.abs()
    assert ((y - u).abs() <= du + U * u.abs()).all()


@pytest.mark.parametrize("shape", [(1, 512, 8, 8), (1, 64, 60, 80), (300, 200), (64, 4096), (3, 258, 31, 37), (4, 9000), (16, 70, 7, 9)])
def test_no_further_from_64_bits_than_elementary_operations(dev, shape):
    """The root mean square distance of y and dx from 64 bits, against the same formulas as elementary fp32 operations: a value here passes
    through one rounding fewer (x - mean, its product with rstd less the correction, the product with the weight plus the bias)."""
    from taming_event_flow_amd.models.norm import layer_norm

    C, lane = shape[1], [1, -1] + [1] * (len(shape) - 2)
    ours, plains = [0.0, 0.0], [0.0, 0.0]
    for seed in range(3):
        gen = torch.Generator(device=dev).manual_seed(seed)
        x = torch.randn(shape, generator=gen, device=dev) * 2 + 0.3
        w, b = 1 + 0.2 * torch.randn(C, generator=gen, device=dev), 0.1 * torch.randn(C, generator=gen, device=dev)
        dy = torch.randn(shape, generator=gen, device=dev)

        def formulas(x, w, b, dy):
            w, b = w.view(lane), b.view(lane)
            d = x - x.mean(1, keepdim=True)
            rstd = 1 / ((d * d).mean(1, keepdim=True) + 1e-5).sqrt()
            u, h = d * rstd, dy * w
            return u * w + b, rstd * (h - h.mean(1, keepdim=True) - u * (h * u).mean(1, keepdim=True))

        xl = x.clone().requires_grad_(True)
        y = layer_norm(xl, w, b)
        got = (y.detach(), torch.autograd.grad(y, xl, dy)[0])
        want = formulas(x.double(), w.double(), b.double(), dy.double())
        plain = formulas(x, w, b, dy)
        for i in range(2):
            ours[i] += (got[i] - want[i]).square().sum().item()
            plains[i] += (plain[i] - want[i]).square().sum().item()
    assert ours[0] <= plains[0] and ours[1] <= plains[1], [(a / p) ** 0.5 for a, p in zip(ours, plains)]
