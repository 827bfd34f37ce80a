"""Orthogonalisation of matrices of up to 8 rows (or columns), whose sums and iteration are 64 bits: rounded once, at the end.

Tolerances.  U = 2^-24 is half a step of fp32, E = 2^-53 of fp64.  Five steps: A = X X^T carries some 16 roundings of E, the
iteration on A multiplies them by up to a^2 a step, and they reach the result through b A: 16 E |b| a^10 = 2e-9 of the largest element, besides
U |value| (half a step of the type where that is a 16-bit one).
More steps, against an iteration in 80 bits: A is summed again before its roundings have grown by more than 1e6, so the same term is
16 E |b| min(a^(2 steps), 1e6) whatever the number of steps; and 32 roundings a step of X; along a singular value s they grow until it has reached the size of 1, by 1 / s,
and by a a step where s is 0 (then only while 16 E a^steps is below 1e-6; beyond, the result's singular values stay where the polynomial puts
values of that size: below 1.3)."""
import ctypes

import numpy as np
import pytest
import torch
from test_ortho_gpu import ABC, dev, iterate, matrix  # noqa: F401

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -24, 2.0 ** -53
SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (4, 4), (8, 8), (5, 64), (65, 5), (7, 1000), (8, 1024), (1024, 8), (8, 1025), (8, 2048), (3, 5000), (5000, 3), (2, 70001), (1, 300000)]
KINDS = ["normal", "rank", "deficient", "decay", "rows", "equal"]


def close(got, u, want):
    want = want.double()
    T = U if u.dtype == torch.float32 else torch.finfo(u.dtype).eps / 2
    bound = (T + (U if T != U else 0)) * want.abs() + 2e-9 * want.abs().max() + T * torch.finfo(u.dtype).smallest_normal
    err = (got.detach().double().cpu() - want).abs()
    assert got.shape == u.shape and got.dtype == u.dtype and (err <= bound).all(), (tuple(u.shape), (err - bound).max().item())


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", KINDS)
def test_rounded_once(dev, shape, kind):  # noqa: F811
    from taming_event_flow_amd.optim import orthogonalize

    u = matrix(kind, *shape, seed=sum(shape)).float().to(dev)
    close(orthogonalize(u), u, iterate(u, 5, ABC, 1e-7, torch.float64))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 3), (8, 700), (2500, 5), (3, 9000)])
def test_half_types(dev, dtype, shape):  # noqa: F811
    from taming_event_flow_amd.optim import orthogonalize

    u = matrix("rank", *shape, seed=1).to(dtype).to(dev)
    close(orthogonalize(u), u, iterate(u, 5, ABC, 1e-7, torch.float64))


def iterate80(u, steps, abc):
    x = u.cpu().numpy().astype(np.longdouble)
    x = x / np.sqrt((x * x).sum())
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    a, b, c = (np.longdouble(v) for v in abc)
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return torch.from_numpy(np.ascontiguousarray(x.T if tall else x).astype(np.float64))


@pytest.mark.parametrize("steps", [1, 4, 8, 9, 16, 24, 32])
@pytest.mark.parametrize("abc", [ABC, (2.0, -1.5, 0.5), (1.5, -0.5, 0.0)])
@pytest.mark.parametrize("kind", KINDS)
def test_many_steps(dev, steps, abc, kind):  # noqa: F811
    from taming_event_flow_amd.optim import orthogonalize

    for shape in ((2, 3), (8, 40), (300, 5), (4, 2500)):
        u = matrix(kind, *shape, seed=steps).float().to(dev)
        y = orthogonalize(u, steps=steps, coefficients=abc).double().cpu()
        s = torch.linalg.svdvals(u.double().cpu())
        lowest = (s[-1] / torch.linalg.vector_norm(s)).item()
        grown = min(32 * steps / max(lowest, 1e-300), 16 * abc[0] ** steps) * E
        if lowest > 1e-5 or grown < 1e-6:
            want = iterate80(u, steps, abc)
            bound = U * want.abs() + (grown + 16 * E * abs(abc[1]) * min(abc[0] ** (2 * steps), 1e6)) * want.abs().max()
            assert ((y - want).abs() <= bound).all(), (shape, ((y - want).abs() - bound).max().item(), grown)
        assert torch.linalg.matrix_norm(y, 2) < 1.3, shape


@pytest.mark.parametrize("shape", [(2, 3), (8, 500), (6, 4000), (3000, 4)])
def test_zero_nan_inf_stay_in_their_matrix(dev, shape):  # noqa: F811
    from taming_event_flow_amd.optim import orthogonalize

    u = matrix("normal", *shape).float().to(dev).repeat(5, 1, 1)
    for steps in (5, 12):
        v = u.clone()
        clean = orthogonalize(v, steps=steps)
        v[1] = 0
        v[2, 1, 2], v[3, 0, -1] = float("nan"), float("-inf")
        y = orthogonalize(v, steps=steps)
        assert not y[1].any() and torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
        assert torch.equal(y[0], clean[0]) and torch.equal(y[4], clean[4])


def test_alone_in_batches_in_lists(dev):  # noqa: F811
    from taming_event_flow_amd.optim import orthogonalize

    for steps in (5, 10):
        many = [matrix("rank", *s, seed=i).float().to(dev) for i, s in enumerate([(2, 3), (8, 1024), (8, 1025), (3, 9000), (9000, 3), (1, 5), (300, 500)] * 6)]
        alone = [orthogonalize(u, steps=steps) for u in many[:6]]
        got = orthogonalize(many, steps=steps)
        for i, y in enumerate(got):
            if i % 7 < 6:
                base = orthogonalize(many[i], steps=steps) if i >= 7 else alone[i]
                assert torch.equal(y, base), i
        batch = torch.stack([matrix("normal", 5, 3000, seed=k).float() for k in range(4)]).to(dev)
        y = orthogonalize(batch, steps=steps)
        assert all(torch.equal(y[k], orthogonalize(batch[k], steps=steps)) for k in range(4))
        same = batch[0].expand(3, 5, 3000)
        assert all(torch.equal(z, y[0]) for z in orthogonalize(same, steps=steps))


def test_views(dev):  # noqa: F811
    from taming_event_flow_amd.optim import orthogonalize

    wide = torch.full((20, 5000), float("nan"), device=dev)
    for view in (wide[3:9, 5:105], wide[3:9, 7:4000], wide[3:19:3, 5:105], wide[3:9, 5:4000].T):
        view.copy_(matrix("normal", *view.shape, seed=5))
        close(orthogonalize(view), view, iterate(view, 5, ABC, 1e-7, torch.float64))
        view.fill_(float("nan"))


@pytest.mark.parametrize("shape", [(5, 60), (5, 6000), (6000, 5)])
@pytest.mark.parametrize("steps", [5, 12])
def test_in_place(dev, shape, steps):  # noqa: F811
    """The library's entry point may be given the matrix itself for the result."""
    from taming_event_flow_amd import _lib
    from taming_event_flow_amd.optim import orthogonalize

    u = matrix("normal", *shape).float().to(dev)
    want = orthogonalize(u, steps=steps)
    rows, cols = shape
    lib = _lib.lib()
    arr = (_lib.OrthoMatrix * 1)(_lib.OrthoMatrix(u.data_ptr(), u.data_ptr(), rows, cols, cols, cols, 1, 0, 0))
    n = lib.tef_orthogonalize_workspace_bytes(arr, 1)
    ws = torch.empty(n + 255, dtype=torch.uint8, device=dev)
    _lib.check(lib.tef_orthogonalize(arr, 1, 0, steps, *ABC, 1e-7, (ws.data_ptr() + 255) & ~255, n, _lib.stream_ptr()), "in place")
    assert torch.equal(u, want)


def test_workspace_is_what_is_used(dev):  # noqa: F811
    """Bytes behind the workspace that was asked for stay as they are."""
    from taming_event_flow_amd import _lib

    lib = _lib.lib()
    for shapes in ([(8, 2049)], [(3, 200000), (200000, 3)], [(2, 5000)] * 20):
        us = [torch.randn(s, device=dev) for s in shapes]
        out = [torch.empty_like(u) for u in us]
        arr = (_lib.OrthoMatrix * len(us))(*[_lib.OrthoMatrix(u.data_ptr(), o.data_ptr(), *u.shape, u.shape[1], u.shape[1], 1, 0, 0) for u, o in zip(us, out)])
        n = lib.tef_orthogonalize_workspace_bytes(arr, len(us))
        ws = torch.full((n + 4096,), 77, dtype=torch.uint8, device=dev)
        at = (ws.data_ptr() + 255) & ~255
        _lib.check(lib.tef_orthogonalize(arr, len(us), 0, 12, *ABC, 1e-7, at, n, _lib.stream_ptr()), "workspace")
        assert (ws[at - ws.data_ptr() + n:] == 77).all() and all(torch.isfinite(o).all() for o in out)


def test_graph(dev):  # noqa: F811
    from taming_event_flow_amd.optim import orthogonalize

    u, v = matrix("normal", 6, 50).float().to(dev), matrix("normal", 6, 5000).float().to(dev)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        orthogonalize([u, v], steps=12)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = orthogonalize([u, v], steps=12)
    for k in range(3):
        u.copy_(matrix("rank", 6, 50, seed=k + 10))
        v.copy_(matrix("rank", 6, 5000, seed=k + 20))
        graph.replay()
        torch.cuda.synchronize()
        eager = orthogonalize([u, v], steps=12)
        assert torch.equal(y[0], eager[0]) and torch.equal(y[1], eager[1]), k
