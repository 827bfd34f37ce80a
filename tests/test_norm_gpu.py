"""Layer normalisation (models/norm.py on csrc/tef_norm.hip) against the formulas in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32, r = eps(T) / 2 half a step of the type the result is stored in.  A sum over
the C elements of a row passes through at most D additions (a lane's own elements, then the joins of lanes and waves), so a
mean is off by at most D u mean|x|, which with the rounding of the subtraction puts u = (x - mean) rstd off by
du = D u (mean|x| + |x|) rstd + 2 D u |u| (the second term: the variance's own sum, halved by the square root, and the last
products).  A result below the type's smallest normal number is stored on a grid of fixed steps eps(T) * smallest_normal (2^-24
in fp16), so it is off by half of that whatever its own size: every bound holds r * smallest_normal besides r |value|.
Everything behind it is bounded by the derivative times that, plus a handful of roundings.  The bounds are
per element and computed in 64 bits with the reference itself."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = {None: lambda z: z, "relu": lambda z: z.clamp(min=0), "tanh": torch.tanh, "sigmoid": torch.sigmoid}
SLOPES = {None: torch.ones_like, "relu": lambda z: (z > 0).double(), "tanh": lambda z: 1 - torch.tanh(z) ** 2,
          "sigmoid": lambda z: torch.sigmoid(z) * (1 - torch.sigmoid(z))}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    import __graft_entry__ as g

    g.build()
    return torch.device("cuda:0")


def reference(x, w, b, res, dim, eps, act, dy):
    """Values and bounds of y, dx, dw, db, dres in 64 bits on the CPU (dim moved last and back)."""
    cut = lambda t: t.detach().double().cpu().movedim(dim, -1)  # noqa: E731
    back = lambda t: t.movedim(-1, dim)  # noqa: E731
    T = torch.finfo(x.dtype).eps / 2
    x64, C = cut(x), x.shape[dim]
    rows = x64.numel() // C
    w64 = w.detach().double().cpu() if w is not None else torch.ones(C, dtype=torch.float64)
    b64 = b.detach().double().cpu() if b is not None else torch.zeros(C, dtype=torch.float64)
    r64 = cut(res) if res is not None else torch.zeros_like(x64)
    D = 100 + C / 256
    mean = x64.mean(-1, keepdim=True)
    rstd = 1 / (((x64 - mean) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    u = (x64 - mean) * rstd
    du = D * U * (x64.abs().mean(-1, keepdim=True) + x64.abs()) * rstd + 2 * D * U * u.abs()
    z = u * w64 + b64 + r64
    dz = du * w64.abs() + 4 * U * ((u * w64).abs() + b64.abs() + r64.abs())
    y = ACTS[act](z)
    tiny = torch.finfo(x.dtype).smallest_normal
    out = {"y": (back(y), back(dz + 8 * U * y.abs() + T * y.abs() + T * tiny))}
    if dy is None:
        return out, z, dz
    d64 = cut(dy)
    g = d64 * SLOPES[act](z)
    dg = (d64.abs() * dz if act in ("tanh", "sigmoid") else 0) + 16 * U * d64.abs()      # |act''| < 1
    h, dh = g * w64, dg * w64.abs() + 2 * U * (g * w64).abs()
    s1, s2 = h.mean(-1, keepdim=True), (h * u).mean(-1, keepdim=True)
    ds1 = dh.mean(-1, keepdim=True) + D * U * h.abs().mean(-1, keepdim=True)
    ds2 = (dh * u.abs() + h.abs() * du).mean(-1, keepdim=True) + D * U * (h * u).abs().mean(-1, keepdim=True)
    dx = rstd * (h - s1 - u * s2)
    drs = D * U * (1 + 2 * x64.abs().mean(-1, keepdim=True) * rstd)      # rstd itself, relative
    ddx = rstd * (dh + ds1 + du * s2.abs() + u.abs() * ds2 + 4 * U * (h.abs() + s1.abs() + (u * s2).abs())) + drs * dx.abs()
    out["dx"] = (back(dx), back(ddx + T * dx.abs() + T * tiny))
    out["dres"] = (back(g), back(dg + T * g.abs() + T * tiny))
    Dw, flat = 100 + rows / 256, tuple(range(x64.dim() - 1))
    Tw = torch.finfo(w.dtype).eps / 2 if w is not None else U
    tiny_w = Tw * torch.finfo(w.dtype if w is not None else torch.float32).smallest_normal
    dw, db = (g * u).sum(flat), g.sum(flat)
    gu, ga = (g * u).abs().sum(flat), g.abs().sum(flat)
    edg = dg if torch.is_tensor(dg) else torch.zeros_like(g)
    out["dw"] = (dw, (edg * u.abs() + g.abs() * du).sum(flat) + Dw * U * gu + Tw * dw.abs() + tiny_w)
    out["db"] = (db, edg.sum(flat) + Dw * U * ga + Tw * db.abs() + tiny_w)
    return out, z, dz


def check(name, got, want):
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), (name, got.shape, value.shape)
    if value.numel() == 0:
        return
    err = (got.detach().double().cpu() - value).abs()
    worst = (err / bound.clamp(min=1e-300)).max().item()
    assert torch.isfinite(got).all() and worst <= 1.0, (name, worst, err.max().item(), value.abs().max().item())


def make(shape, dim, dtype, wdtype, dev, seed=0, residual=False, affine=True, offset=0.5):
    gen = torch.Generator().manual_seed(seed)
    C = shape[dim]
    x = (torch.randn(shape, generator=gen) * 2 + offset).to(dtype).to(dev)
    w = (1 + 0.3 * torch.randn(C, generator=gen)).to(wdtype).to(dev) if affine else None
    b = (0.2 * torch.randn(C, generator=gen)).to(wdtype).to(dev) if affine else None
    r = torch.randn(shape, generator=gen).to(dtype).to(dev) if residual else None
    dy = torch.randn(shape, generator=gen).to(dtype).to(dev)
    return x, w, b, r, dy


def run_both(x, w, b, r, dy, dim, eps, act):
    from taming_event_flow_amd.models.norm import layer_norm

    leaves = {"dx": x, "dw": w, "db": b, "dres": r}
    leaves = {k: t.detach().requires_grad_(True) for k, t in leaves.items() if t is not None}
    y = layer_norm(leaves["dx"], leaves.get("dw"), leaves.get("db"), dim, eps, act, leaves.get("dres"))
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    want, z, dz = reference(x, w, b, r, dim, eps, act, dy)
    if act == "relu":      # (a case whose z lies closer to 0 than its own error has no gradient to compare)
        assert (z.abs() > dz).all()
    check("y", y, want["y"])
    for k, g in zip(leaves, grads):
        assert g.dtype == leaves[k].dtype
        check(k, g, want[k])
    return y, grads


# rows: one lane, a part of a wave, a wave, several packs a lane, the workgroup forms and the long form, odd everywhere
ROWS = [(1, 1), (3, 1), (5, 2), (257, 3), (1, 18), (33, 64), (7, 255), (2, 256), (3, 257), (5, 1030), (2, 2048), (3, 2049),
        (2, 4099), (2, 8192), (3, 8193), (1, 40001)]
# maps: positions in fours and singly, channel counts at and past a power of two, past the registers, one position
MAPS = [(1, 1, 2, 2), (2, 3, 5, 7), (1, 512, 8, 8), (3, 64, 4, 4), (2, 258, 3, 5), (1, 64, 1, 3), (2, 17, 31, 1), (1, 1030, 2, 2),
        (1, 1024, 2, 2), (2, 1100, 1, 3), (1, 5000, 1, 3), (4, 32, 40, 40), (1, 100, 33, 64)]


@pytest.mark.parametrize("shape", ROWS + MAPS)
def test_sizes(dev, shape):
    dim = 1
    x, w, b, r, dy = make(shape, dim, torch.float32, torch.float32, dev, seed=sum(shape))
    run_both(x, w, b, r, dy, dim, 1e-5, None)


@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.float16, torch.float16),
                                          (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("act", [None, "tanh", "sigmoid"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(37, 130), (2, 2500), (3, 40, 6, 6), (2, 66, 5, 3), (1, 9000)])
def test_types_activations_residual(dev, dtype, wdtype, act, residual, shape):
    x, w, b, r, dy = make(shape, 1, dtype, wdtype, dev, seed=7, residual=residual)
    run_both(x, w, b, r, dy, 1, 1e-5, act)


@pytest.mark.parametrize("shape", [(6, 31), (2, 8, 3, 4), (1, 5, 3, 3)])
@pytest.mark.parametrize("residual", [False, True])
def test_relu(dev, shape, residual):
    x, w, b, r, dy = make(shape, 1, torch.float32, torch.float32, dev, seed=11, residual=residual)
    run_both(x, w, b, r, dy, 1, 1e-5, "relu")


@pytest.mark.parametrize("dim", [0, 1, 2, 3, -1, -2])
def test_every_dimension(dev, dim):
    x, w, b, r, dy = make((3, 4, 5, 6), dim, torch.float32, torch.float32, dev, seed=3)
    run_both(x, w, b, r, dy, dim, 1e-3, "tanh")


def test_layouts(dev):
    """Channels-last maps, every second column, a start one element into the storage, an expanded gradient and a transposed
    residual give what the contiguous tensors give; the result has x's memory order."""
    from taming_event_flow_amd.models.norm import layer_norm

    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, r, dy = make((2, 24, 6, 10), 1, dtype, torch.float32, dev, seed=5, residual=True)
        want, _, _ = reference(x, w, b, r, 1, 1e-5, "tanh", dy)
        cl = lambda t: t.contiguous(memory_format=torch.channels_last)  # noqa: E731
        wide = torch.zeros((2, 24, 6, 20), dtype=dtype, device=dev)
        wide[..., ::2] = x
        store = torch.zeros(x.numel() + 1, dtype=dtype, device=dev)
        store[1:] = x.reshape(-1)
        turned = r.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)
        for xv, rv, dv in ((cl(x), r, dy), (cl(x), cl(r), cl(dy)), (wide[..., ::2], turned, dy), (store[1:].view(x.shape), r, cl(dy))):
            xl, rl = xv.detach().requires_grad_(True), rv.detach().requires_grad_(True)
            y = layer_norm(xl, w, b, activation="tanh", residual=rl)
            dx, dr = torch.autograd.grad(y, (xl, rl), dv)
            check("y", y, want["y"]), check("dx", dx, want["dx"]), check("dres", dr, want["dres"])
        assert layer_norm(cl(x), w, b).is_contiguous(memory_format=torch.channels_last)
        one = torch.ones((), dtype=dtype, device=dev).expand(x.shape)
        want, _, _ = reference(x, w, b, None, 1, 1e-5, None, one)
        xl = x.detach().requires_grad_(True)
        layer_norm(xl, w, b).backward(one)
        check("dx", xl.grad, want["dx"])


def test_parts_missing(dev):
    """No weight, no bias, neither; gradients of some leaves only."""
    from taming_event_flow_amd.models.norm import layer_norm

    for shape in ((9, 50), (2, 12, 3, 4)):
        x, w, b, r, dy = make(shape, 1, torch.float32, torch.float32, dev, seed=2, residual=True)
        for wv, bv in ((None, None), (w, None), (None, b)):
            want, _, _ = reference(x, wv, bv, r, 1, 1e-5, "sigmoid", dy)
            xl = x.detach().requires_grad_(True)
            y = layer_norm(xl, wv, bv, activation="sigmoid", residual=r)
            check("y", y, want["y"])
            check("dx", torch.autograd.grad(y, xl, dy)[0], want["dx"])
        want, _, _ = reference(x, w, b, r, 1, 1e-5, "tanh", dy)
        for which in ("dw", "db", "dres"):
            leaf = {"dw": w, "db": b, "dres": r}[which].detach().requires_grad_(True)
            args = {"dw": w, "db": b, "dres": r, which: leaf}
            y = layer_norm(x, args["dw"], args["db"], activation="tanh", residual=args["dres"])
            check(which, torch.autograd.grad(y, leaf, dy)[0], want[which])
        with torch.no_grad():
            check("y", layer_norm(x, w, b, activation="tanh", residual=r), want["y"])


def test_gradient_against_differences(dev):
    """The gradient of <dy, y> along a random direction of every argument against a central difference in 64 bits."""
    from taming_event_flow_amd.models.norm import layer_norm

    x, w, b, r, dy = make((3, 10, 2, 4), 1, torch.float32, torch.float32, dev, seed=9, residual=True)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(layer_norm(leaves[0], leaves[1], leaves[2], activation="tanh", residual=leaves[3]), leaves, dy)
    f = lambda a: (reference(*a, 1, 1e-5, "tanh", None)[0]["y"][0] * dy.double().cpu()).sum().item()  # noqa: E731
    gen = torch.Generator().manual_seed(1)
    args = [t.double().cpu() for t in (x, w, b, r)]
    for i, g in enumerate(grads):
        v = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        hi = f([a + h * v if j == i else a for j, a in enumerate(args)])
        lo = f([a - h * v if j == i else a for j, a in enumerate(args)])
        slope = (g.double().cpu() * v).sum().item()
        scale = (g.double().cpu() * v).abs().sum().item()
        # the difference: third derivative h^2 / 6 (of order scale * 10) and cancellation 2^-52 / h; the gradient: its fp32 bound
        assert abs((hi - lo) / (2 * h) - slope) <= scale * (200 * U + 1e-8) + 1e-8, i


def test_second_derivative_is_refused(dev):
    from taming_event_flow_amd.models.norm import layer_norm

    x = torch.randn(3, 8, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(layer_norm(x).sum(), x, create_graph=True)


def test_empty(dev):
    from taming_event_flow_amd.models.norm import layer_norm

    w, b = torch.ones(8, device=dev, requires_grad=True), torch.zeros(8, device=dev, requires_grad=True)
    for shape in ((0, 8), (0, 8, 4, 4), (2, 8, 0, 4)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        y = layer_norm(x, w, b)
        assert y.shape == x.shape
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert dx.shape == x.shape and not dw.any() and not db.any()


def test_offset_and_constant_rows(dev):
    """A mean a thousand times the spread costs mean / spread roundings and no more; a constant row gives the bias."""
    from taming_event_flow_amd.models.norm import layer_norm

    for shape in ((4, 300), (2, 48, 4, 4)):
        x, w, b, r, dy = make(shape, 1, torch.float32, torch.float32, dev, seed=4, offset=2000.0)
        run_both(x, w, b, None, dy, 1, 1e-5, None)
        c = torch.full(shape, 3.0, device=dev)
        y = layer_norm(c, w, b)
        assert torch.equal(y, b.view([1, -1] + [1] * (len(shape) - 2)).expand(shape))


def test_non_finite_stay_in_their_row(dev):
    from taming_event_flow_amd.models.norm import layer_norm

    x, w, b, _, _ = make((6, 40), 1, torch.float32, torch.float32, dev, seed=6)
    clean = layer_norm(x, w, b)
    x[1, 3], x[4, 0] = float("nan"), float("inf")
    y = layer_norm(x, w, b, activation="relu")
    assert torch.isnan(y[1]).all() and torch.isnan(y[4]).all()
    for k in (0, 2, 3, 5):
        assert torch.equal(y[k], clean[k].clamp(min=0))
    m = torch.randn((1, 40, 2, 3), device=dev)
    clean = layer_norm(m, w, b)
    m[0, 5, 1, 1] = float("-inf")
    y = layer_norm(m, w, b)
    bad = torch.isnan(y[0]).all(0)
    assert bad[1, 1] and bad.sum() == 1 and torch.equal(y[0][:, ~bad], clean[0][:, ~bad])


def test_reproducible_other_stream_and_graph(dev):
    """Bit for bit the same result again, on a side stream, and from a replayed graph whose input changes."""
    from taming_event_flow_amd.models.norm import layer_norm

    for shape in ((5000, 96), (6, 64, 32, 32)):
        x, w, b, r, dy = make(shape, 1, torch.float32, torch.float32, dev, seed=8, residual=True)

        def step(x_, dy_):
            leaves = [t.detach().requires_grad_(True) for t in (x_, w, b, r)]
            y = layer_norm(leaves[0], leaves[1], leaves[2], activation="tanh", residual=leaves[3])
            return [y.detach()] + list(torch.autograd.grad(y, leaves, dy_))

        first = step(x, dy)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(x, dy)
            sx, sdy = x.clone(), dy.clone()
            step(sx, sdy)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(first, other))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step(sx, sdy)
        for k in range(3):
            sx.copy_(x + k), sdy.copy_(dy * (k + 1))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(step(x + k, dy * (k + 1)), captured)), k


def test_offsets_past_32_bits(dev):
    """More than 2^31 elements: the last rows / positions of a tensor whose offsets need 64 bits."""
    from taming_event_flow_amd.models.norm import layer_norm

    for shape, tail in (((70001, 32768), lambda t: t[-3:]), ((33, 1024, 256, 257), lambda t: t[-1:, :, -2:])):
        C = shape[1]
        x = torch.zeros(shape, dtype=torch.bfloat16, device=dev)
        part = torch.randn(tail(x).shape, device=dev).to(x.dtype)
        tail(x).copy_(part)
        w, b = torch.linspace(0.5, 1.5, C, device=dev), torch.linspace(-1, 1, C, device=dev)
        y = layer_norm(x, w, b)
        want, _, _ = reference(part, w, b, None, 1, 1e-5, None, None)
        check("y", tail(y), want["y"])
        assert torch.equal(y[0].movedim(0, -1).reshape(-1, C)[0], b.to(x.dtype))
        del x, y


def test_module_and_layers(dev):
    """norm="LN" in the network's layers: convolution, normalisation, activation — forward and every gradient against the same
    layers put together in 64 bits."""
    import torch.nn.functional as F

    from taming_event_flow_amd.models.submodules import ConvLayer, ResidualBlock, UpsampleConvLayer

    def norm64(m, t):
        mu = t.mean(1, keepdim=True)
        s = ((t - mu) ** 2).mean(1, keepdim=True)
        v = [1, -1, 1, 1]
        return (t - mu) / (s + m.eps).sqrt() * m.weight.view(v) + m.bias.view(v)

    def conv64(c, t, stride=1):
        return F.conv2d(t, c.weight, c.bias, stride=stride, padding=c.kernel_size[0] // 2)

    torch.manual_seed(0)
    cases = [(ConvLayer(5, 12, 3, 2, "tanh", norm="LN"), (2, 5, 8, 12), lambda m, t: torch.tanh(norm64(m.norm_layer, conv64(m.conv2d, t, 2)))),
             (ResidualBlock(8, 8, activation="tanh", norm="LN"), (2, 8, 6, 6), lambda m, t: torch.tanh(
                 norm64(m.norm2, conv64(m.conv2, torch.tanh(norm64(m.norm1, conv64(m.conv1, t))))) + t)),
             (UpsampleConvLayer(6, 7, 3, activation="sigmoid", norm="LN"), (1, 6, 4, 5), lambda m, t: torch.sigmoid(
                 norm64(m.norm_layer, conv64(m.conv2d, F.interpolate(t, scale_factor=2, mode="bilinear", align_corners=False)))))]
    for layer, shape, plain in cases:
        import copy

        for p in layer.parameters():
            torch.nn.init.normal_(p, 0.3, 0.4)
        twin = copy.deepcopy(layer).double()
        layer = layer.to(dev)
        x = torch.randn(shape)
        xl, x64 = x.to(dev).requires_grad_(True), x.double().requires_grad_(True)
        y = layer(xl)
        y = y[0] if isinstance(y, tuple) else y
        y64 = plain(twin, x64)
        dy = torch.randn(y64.shape, dtype=torch.float64)
        got = torch.autograd.grad(y, [xl] + list(layer.parameters()), dy.float().to(dev))
        want = torch.autograd.grad(y64, [x64] + list(twin.parameters()), dy.float().double())
        # convolutions of up to 72 products summed in fp32, normalised, twice at most: 1e-4 of the largest value, the package's bar
        for g, v in [(y, y64)] + list(zip(got, want)):
            assert (g.detach().double().cpu() - v).abs().max() <= 1e-4 * max(v.abs().max().item(), 1e-3 * dy.abs().sum().item() ** 0.5), type(layer)
