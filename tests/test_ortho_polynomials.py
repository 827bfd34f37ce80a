"""Which coefficients the orthogonalisation and its optimiser take: the same, and asked for before anything is counted or launched."""
import pytest
import torch

ABC = (3.4445, -4.7750, 2.0315)
TAKEN = [ABC, (4.0848, -6.8946, 2.9270), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0), (-1.5, 0.5, 0.0)]
REFUSED = [(16.0, 0.0, 0.0), (4.0, 0.0, 0.0), (0.0, 0.0, 5.0), (-20.0, 0.0, 0.0), (8.5, -20.0, 13.0), (1.0, 40.0, 0.0), (3.9, -6.0, 2.6)]


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as g

    g.build()
    from taming_event_flow_amd import _lib

    return _lib.lib()


def test_check(lib):
    for abc in TAKEN:
        assert lib.tef_orthogonalize_check(5, *abc, 1e-7) == 0, abc
    for abc in REFUSED:
        assert lib.tef_orthogonalize_check(5, *abc, 1e-7) == -1 and b"coefficients" in lib.tef_last_error(), abc
    assert lib.tef_orthogonalize_check(0, *ABC, 1e-7) == -1 and lib.tef_orthogonalize_check(33, *ABC, 1e-7) == -1
    assert lib.tef_orthogonalize_check(5, *ABC, 0.0) == -1 and lib.tef_orthogonalize_check(5, float("nan"), 0.0, 0.0, 1e-7) == -1


def test_optimiser_refuses_when_it_is_made(lib):
    from taming_event_flow_amd import optim, parallel

    bucket = parallel.FlatGradBucket([torch.nn.Parameter(torch.zeros(4, 6))])
    for abc in REFUSED:
        with pytest.raises(ValueError, match="coefficients"):
            optim.FusedMuon(bucket, 0.1, coefficients=abc)
    for abc in TAKEN:      # (the next check is the device's)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            optim.FusedMuon(bucket, 0.1, coefficients=abc)
