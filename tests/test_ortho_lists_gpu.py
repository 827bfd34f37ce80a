"""Newton-Schulz orthogonalisation of lists: what a matrix comes out as does not depend on what is beside it."""
import pytest
import torch
from test_ortho_gpu import check, dev, matrix  # noqa: F401

pytestmark = pytest.mark.gpu


def test_small_matrices_alone_and_in_a_list(dev):  # noqa: F811
    """One-workgroup matrices of both kinds, alone, together, and beside ones that go through tiles: the same bits."""
    from taming_event_flow_amd.optim import orthogonalize

    shapes = [(2, 3), (8, 100), (7, 9), (40, 60), (64, 320), (300, 64), (3, 3), (1, 960), (9, 9)]
    small = [matrix("rank", *s, seed=i).float().to(dev) for i, s in enumerate(shapes)]
    large = [matrix("rank", *s, seed=i).float().to(dev) for i, s in enumerate([(300, 500), (65, 65), (64, 1152)])]
    alone = [orthogonalize(u) for u in small]
    for many in (small, small + large, [large[0]] + small + large[1:], small * 9 + large):
        for g, u in zip(orthogonalize(many), many):
            which = [i for i, s in enumerate(small) if s is u]
            if which:
                assert torch.equal(g, alone[which[0]]), (shapes[which[0]], len(many))
            else:
                check(g, u)
